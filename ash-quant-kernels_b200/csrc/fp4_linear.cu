// Products with 4-bit operands: which kernel takes one, and the W4A4 linear layer, whose x arrives in 16 bits and is
// quantised on the way.
#include <atomic>

#include "fp4.cuh"

namespace ashqk {
namespace {

std::atomic<int> g_matmul_kernel{0};
constexpr int kMaxRows = 1 << 30;  // of either operand: tile coordinates are 32-bit

// Few rows go to the rows kernel, whose CTAs split K, the others to CTA pairs. Measured in graphs (MXFP4, us, rows
// against pairs): 64 rows 8.1 / 9.2 (4096->6144), 8.0 / 9.0 (4096->4096), 10.7 / 14.5 (12288->4096), 14.4 / 17.2
// (4096->24576); 128 rows 9.8 / 9.7, 8.7 / 9.4, 12.7 / 14.8, 16.7 / 18.1; 256 rows 10.0 / 9.7, 10.2 / 9.5, 16.8 / 14.8,
// 28.2 / 18.4. Between 64 and 128 rows only layers of few tiles, whose K is split finely, take the rows kernel. The wide
// layer would gain from it too (8 % at 128 rows); where between 6144 and 24576 that begins was not measured.
bool few_rows(int M, int N) { return M <= 64 || (M <= 128 && N <= 5120); }

int fp4_matmul(const Fp4Product& p, cudaStream_t stream) {
  const int which = g_matmul_kernel.load(std::memory_order_relaxed);
  const bool rows = which ? which == 1 : few_rows(p.a.rows, p.b.rows);
  return rows ? fp4_matmul_rows(p, stream) : fp4_matmul_pair(p, stream);
}

// Q(x) in the workspace: scales first (a multiple of 512 bytes), then codes.
void workspace_layout(int M, int K, int format, size_t* codes_offset, size_t* bytes) {
  *codes_offset = static_cast<size_t>(ceil_div64(M, kFp4TileRows) * fp4_scale_tiles(K, format) * kFp4TileBytes);
  *bytes = *codes_offset + static_cast<size_t>(M) * (fp4_padded_k(K) / 2);
}

int check_product(const void* y, int64_t y_ld, int dtype, int M, int N, int K, int format) {
  if (!y || M <= 0 || N <= 0 || K <= 0 || K > kFp4MaxK || y_ld < N || !fp4_format_ok(format))
    return ASHQK_ERR_INVALID_ARGUMENT;
  if ((dtype != ASHQK_F16 && dtype != ASHQK_BF16) || !aligned(y, 2)) return ASHQK_ERR_INVALID_ARGUMENT;
  return M > kMaxRows || N > kMaxRows ? ASHQK_ERR_UNSUPPORTED : ASHQK_OK;
}

}  // namespace
}  // namespace ashqk

using namespace ashqk;

extern "C" int ashqk_set_fp4_kernel(int which) {
  if (which < 0 || which > 2) return ASHQK_ERR_INVALID_ARGUMENT;
  g_matmul_kernel.store(which, std::memory_order_relaxed);
  return ASHQK_OK;
}

extern "C" int ashqk_fp4_matmul(const void* a_codes, int64_t a_ld, const void* a_scales, const void* b_codes,
                                int64_t b_ld, const void* b_scales, void* y, int64_t y_ld, int dtype, int M, int N, int K,
                                int format, float alpha, void* stream) {
  if (const int rc = check_product(y, y_ld, dtype, M, N, K, format)) return rc;
  if (const int rc = check_fp4_operand(a_codes, a_ld, a_scales, K)) return rc;
  if (const int rc = check_fp4_operand(b_codes, b_ld, b_scales, K)) return rc;
  const Fp4Matrix a = {static_cast<const uint8_t*>(a_codes), a_ld, static_cast<const uint8_t*>(a_scales), M};
  const Fp4Matrix b = {static_cast<const uint8_t*>(b_codes), b_ld, static_cast<const uint8_t*>(b_scales), N};
  return fp4_matmul({a, b, K, format, alpha, y, y_ld, dtype}, static_cast<cudaStream_t>(stream));
}

extern "C" int ashqk_w4a4_workspace_size(int M, int N, int K, int format, int gated, size_t* bytes) {
  if (!bytes || M <= 0 || N <= 0 || K <= 0 || K > kFp4MaxK || !fp4_format_ok(format)) return ASHQK_ERR_INVALID_ARGUMENT;
  size_t offset;
  *bytes = 0;
  if (!fp4_fused_ok(M, N, K, gated != 0)) workspace_layout(M, K, format, &offset, bytes);
  return ASHQK_OK;
}

extern "C" int ashqk_w4a4_linear(const void* x, int64_t x_ld, int dtype, int gated, float x_scale, const void* w_codes,
                                 int64_t w_ld, const void* w_scales, float w_scale, void* y, int64_t y_ld, int M, int N,
                                 int K, int format, void* workspace, size_t workspace_bytes, void* stream) {
  if (const int rc = check_product(y, y_ld, dtype, M, N, K, format)) return rc;
  if (!x || !aligned(x, 2) || x_ld < static_cast<int64_t>(K) * (gated ? 2 : 1)) return ASHQK_ERR_INVALID_ARGUMENT;
  if (!fp4_global_scale_ok(format, x_scale) || !fp4_global_scale_ok(format, w_scale)) return ASHQK_ERR_INVALID_ARGUMENT;
  if (const int rc = check_fp4_operand(w_codes, w_ld, w_scales, K)) return rc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const Fp4Source src = {x, x_ld, dtype, gated != 0, x_scale};
  const Fp4Matrix w = {static_cast<const uint8_t*>(w_codes), w_ld, static_cast<const uint8_t*>(w_scales), N};
  Fp4Product p = {{nullptr, 0, nullptr, M}, w, K, format, x_scale * w_scale, y, y_ld, dtype};
  if (fp4_fused_ok(M, N, K, src.gated)) return fp4_linear_rows(src, p, st);
  size_t offset, bytes;
  workspace_layout(M, K, format, &offset, &bytes);
  if (!workspace || workspace_bytes < bytes || !aligned(workspace, 16)) return ASHQK_ERR_WORKSPACE;
  uint8_t* scales = static_cast<uint8_t*>(workspace);
  uint8_t* codes = scales + offset;
  const int64_t ld = fp4_padded_k(K) / 2;
  if (const int rc = quantize_fp4(src, codes, ld, scales, M, K, format, true, st)) return rc;
  p.a = {codes, ld, scales, M};
  return fp4_matmul(p, st);
}
