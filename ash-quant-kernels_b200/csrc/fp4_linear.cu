// W4A4 linear layer: x in 16 bits, quantised on the way into the product with 4-bit weights.
#include <atomic>

#include "fp4.cuh"

namespace ashqk {

int dtype_size(int dtype);
int check_fp4_operand(const void* codes, int64_t codes_ld, const void* scales, int K);
bool fp4_global_scale_ok(int format, float gs);
int quantize_fp4(const void* x, int64_t x_ld, int dtype, bool gated, void* codes, int64_t codes_ld, void* scales, int M,
                 int K, int format, float gs, bool early, cudaStream_t stream);

int fp4_matmul_rows(const void* a_codes, int64_t a_ld, const void* a_scales, const void* b_codes, int64_t b_ld,
                    const void* b_scales, void* y, int64_t y_ld, int dtype, int M, int N, int K, int format, float alpha,
                    cudaStream_t stream);
int fp4_matmul_pair(const void* a_codes, int64_t a_ld, const void* a_scales, const void* b_codes, int64_t b_ld,
                    const void* b_scales, void* y, int64_t y_ld, int dtype, int M, int N, int K, int format, float alpha,
                    cudaStream_t stream);

bool fp4_fused_ok(int M, int N, int K);
int fp4_linear_rows(const void* x, int64_t x_ld, int dtype, bool gated, float x_gs, const void* w_codes, int64_t w_ld,
                    const void* w_scales, void* y, int64_t y_ld, int M, int N, int K, int format, float alpha,
                    cudaStream_t stream);

namespace {

std::atomic<int> g_matmul_kernel{0};
constexpr int kMaxRows = 1 << 30;  // of either operand: tile coordinates are 32-bit

// Few rows go to the rows kernel, whose CTAs split K, the others to CTA pairs. Measured in graphs (MXFP4, us, rows
// against pairs): 64 rows 8.2 / 9.4 (4096->6144), 7.9 / 9.1 (4096->4096), 10.9 / 14.9 (12288->4096), 15.2 / 17.6
// (4096->24576); 128 rows 10.5 / 9.9, 9.0 / 9.6, 13.8 / 15.2, 17.6 / 18.7; 256 rows 10.9 / 9.9, 10.8 / 9.6,
// 18.2 / 15.2. Between 64 and 128 rows it is the number of tiles that decides: the fewer, the finer the split of K.
bool few_rows(int M, int N) { return M <= 64 || (M <= 128 && N <= 5120); }

// Q(x) in the workspace: scales first (a multiple of 512 bytes), then codes.
void workspace_layout(int M, int K, int format, size_t* codes_offset, size_t* bytes) {
  *codes_offset = static_cast<size_t>(ceil_div64(M, kFp4TileRows) * fp4_scale_tiles(K, format) * kFp4TileBytes);
  *bytes = *codes_offset + static_cast<size_t>(M) * (fp4_padded_k(K) / 2);
}

}  // namespace
}  // namespace ashqk

using namespace ashqk;

extern "C" int ashqk_set_fp4_kernel(int which) {
  if (which < 0 || which > 2) return ASHQK_ERR_INVALID_ARGUMENT;
  g_matmul_kernel.store(which, std::memory_order_relaxed);
  return ASHQK_OK;
}

extern "C" int ashqk_fp4_matmul(const void* a_codes, int64_t a_ld, const void* a_scales, const void* b_codes, int64_t b_ld,
                                const void* b_scales, void* y, int64_t y_ld, int dtype, int M, int N, int K, int format,
                                float alpha, void* stream) {
  if (!y || M <= 0 || N <= 0 || K <= 0 || K > kFp4MaxK || y_ld < N || !fp4_format_ok(format)) return ASHQK_ERR_INVALID_ARGUMENT;
  if ((dtype != ASHQK_F16 && dtype != ASHQK_BF16) || !aligned(y, 2)) return ASHQK_ERR_INVALID_ARGUMENT;
  if (M > kMaxRows || N > kMaxRows) return ASHQK_ERR_UNSUPPORTED;
  if (const int rc = check_fp4_operand(a_codes, a_ld, a_scales, K)) return rc;
  if (const int rc = check_fp4_operand(b_codes, b_ld, b_scales, K)) return rc;
  const int which = g_matmul_kernel.load(std::memory_order_relaxed);
  const bool pair = which ? which == 2 : !few_rows(M, N);
  return (pair ? fp4_matmul_pair : fp4_matmul_rows)(a_codes, a_ld, a_scales, b_codes, b_ld, b_scales, y, y_ld, dtype, M, N,
                                                    K, format, alpha, static_cast<cudaStream_t>(stream));
}

extern "C" int ashqk_w4a4_workspace_size(int M, int N, int K, int format, size_t* bytes) {
  if (!bytes || M <= 0 || N <= 0 || K <= 0 || K > kFp4MaxK || !fp4_format_ok(format)) return ASHQK_ERR_INVALID_ARGUMENT;
  size_t offset;
  *bytes = 0;
  if (!fp4_fused_ok(M, N, K)) workspace_layout(M, K, format, &offset, bytes);
  return ASHQK_OK;
}

extern "C" int ashqk_w4a4_linear(const void* x, int64_t x_ld, int dtype, int gated, float x_scale, const void* w_codes,
                                 int64_t w_ld, const void* w_scales, float w_scale, void* y, int64_t y_ld, int M, int N,
                                 int K, int format, void* workspace, size_t workspace_bytes, void* stream) {
  if (!x || !y || M <= 0 || N <= 0 || K <= 0 || K > kFp4MaxK || !fp4_format_ok(format)) return ASHQK_ERR_INVALID_ARGUMENT;
  if ((dtype != ASHQK_F16 && dtype != ASHQK_BF16) || !aligned(x, 2) || !aligned(y, 2)) return ASHQK_ERR_INVALID_ARGUMENT;
  if (x_ld < static_cast<int64_t>(K) * (gated ? 2 : 1) || y_ld < N) return ASHQK_ERR_INVALID_ARGUMENT;
  if (!fp4_global_scale_ok(format, x_scale) || !fp4_global_scale_ok(format, w_scale)) return ASHQK_ERR_INVALID_ARGUMENT;
  if (M > kMaxRows || N > kMaxRows) return ASHQK_ERR_UNSUPPORTED;
  if (const int rc = check_fp4_operand(w_codes, w_ld, w_scales, K)) return rc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (fp4_fused_ok(M, N, K))
    return fp4_linear_rows(x, x_ld, dtype, gated != 0, x_scale, w_codes, w_ld, w_scales, y, y_ld, M, N, K, format,
                           x_scale * w_scale, st);
  size_t offset, bytes;
  workspace_layout(M, K, format, &offset, &bytes);
  if (!workspace || workspace_bytes < bytes || !aligned(workspace, 16)) return ASHQK_ERR_WORKSPACE;
  uint8_t* scales = static_cast<uint8_t*>(workspace);
  uint8_t* codes = scales + offset;
  const int64_t ld = fp4_padded_k(K) / 2;
  if (const int rc = quantize_fp4(x, x_ld, dtype, gated != 0, codes, ld, scales, M, K, format, x_scale, true, st)) return rc;
  return ashqk_fp4_matmul(codes, ld, scales, w_codes, w_ld, w_scales, y, y_ld, dtype, M, N, K, format, x_scale * w_scale,
                          stream);
}
