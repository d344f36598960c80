// Thin PyTorch binding over the C ABI in include/ashqk_b200.h.
//
// Registers torch.ops.ashqk.* for the CUDA dispatch key only: a CPU tensor gets
// PyTorch's "could not run ... with arguments from the CPU backend" error, so
// there is no silent host fallback. The binding owns the split-K workspace: one
// zero-initialised byte buffer per (device, stream), grown on demand and left
// zeroed by every kernel -- the role of the reference's _workspace caches
// (ashqk/kernels/w4a16_gemv.py:110-120, ashqk/kernels/w4a16_gemm_v3.py:108-119).
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include <map>
#include <mutex>
#include <tuple>
#include <utility>
#include <vector>

#include "ashqk_b200.h"

namespace {

void check_rc(int rc, const char* what) {
  TORCH_CHECK(rc == ASHQK_OK, "ashqk.", what, ": ", ashqk_status_string(rc), " (status ", rc, ")");
}

std::mutex g_ws_mu;
std::map<std::pair<int, cudaStream_t>, at::Tensor> g_ws;

// Zeroed workspace of at least `bytes` for the current stream of `dev`.
at::Tensor workspace_for(const at::Device& dev, size_t bytes) {
  if (bytes == 0) return at::Tensor();
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  std::lock_guard<std::mutex> lock(g_ws_mu);
  at::Tensor& t = g_ws[{dev.index(), stream}];
  if (!t.defined() || static_cast<size_t>(t.numel()) < bytes) {
    const int64_t rounded = static_cast<int64_t>((bytes + (1u << 20) - 1) >> 20 << 20);
    t = at::zeros({rounded}, at::TensorOptions().dtype(at::kByte).device(dev));
  }
  return t;
}

struct Problem {
  int64_t M, N, K, G;
};

// Shape / dtype / device checks shared by the linear ops. Returns x with a unit
// column stride (a copy only when the caller's x has another inner stride).
Problem check_linear(const at::Tensor& x, const at::Tensor& qw, const at::Tensor& qz, const at::Tensor& s) {
  TORCH_CHECK(x.is_cuda(), "ashqk: x must be a CUDA tensor");
  TORCH_CHECK(x.scalar_type() == at::kHalf && x.dim() == 2, "ashqk: x must be a 2-D float16 tensor");
  TORCH_CHECK(qw.scalar_type() == at::kInt && qw.dim() == 2, "ashqk: qweight must be a 2-D int32 tensor");
  TORCH_CHECK(qz.scalar_type() == at::kInt && qz.dim() == 2, "ashqk: qzeros must be a 2-D int32 tensor");
  TORCH_CHECK(s.scalar_type() == at::kHalf && s.dim() == 2, "ashqk: scales must be a 2-D float16 tensor");
  TORCH_CHECK(qw.device() == x.device() && qz.device() == x.device() && s.device() == x.device(),
              "ashqk: all tensors must be on the same device");
  Problem p;
  p.M = x.size(0);
  p.K = x.size(1);
  p.N = qw.size(1) * 8;
  TORCH_CHECK(s.size(0) > 0 && p.K % s.size(0) == 0, "ashqk: K must be a multiple of scales.shape[0]");
  p.G = p.K / s.size(0);
  TORCH_CHECK(qw.size(0) == p.K, "ashqk: qweight must be [K, N/8]");
  TORCH_CHECK(qz.size(0) == p.K / p.G && qz.size(1) == p.N / 8, "ashqk: qzeros must be [K/G, N/8]");
  TORCH_CHECK(s.size(1) == p.N, "ashqk: scales must be [K/G, N]");
  return p;
}

at::Tensor unit_inner(const at::Tensor& t) { return t.stride(1) == 1 ? t : t.contiguous(); }

enum class Path { kGemv, kGemm, kLinear };

at::Tensor run_linear(Path path, const at::Tensor& x_in, const at::Tensor& qw_in, const at::Tensor& qz_in,
                      const at::Tensor& s_in, int64_t split_k, c10::optional<at::Tensor> out) {
  Problem p = check_linear(x_in, qw_in, qz_in, s_in);
  c10::cuda::CUDAGuard guard(x_in.device());
  at::Tensor x = unit_inner(x_in), qw = unit_inner(qw_in), qz = unit_inner(qz_in), s = unit_inner(s_in);
  at::Tensor y;
  if (out.has_value()) {
    y = *out;
    TORCH_CHECK(y.is_cuda() && y.device() == x.device() && y.scalar_type() == at::kHalf && y.dim() == 2 &&
                    y.size(0) == p.M && y.size(1) == p.N && y.stride(1) == 1,
                "ashqk: out must be a float16 [M, N] CUDA tensor with unit column stride");
  } else {
    y = at::empty({p.M, p.N}, x.options());
  }
  if (p.M == 0) return y;
  TORCH_CHECK(p.M <= INT32_MAX && p.N <= INT32_MAX && p.K <= INT32_MAX, "ashqk: problem too large");
  const int M = static_cast<int>(p.M), N = static_cast<int>(p.N), K = static_cast<int>(p.K),
            G = static_cast<int>(p.G);
  size_t bytes = 0;
  int rc;
  switch (path) {
    case Path::kGemv:
      rc = ashqk_gemv_workspace_size(M < 16 ? M : 16, N, K, G, static_cast<int>(split_k), &bytes);
      break;
    case Path::kGemm:
      rc = ashqk_gemm_workspace_size(M, N, K, G, &bytes);
      break;
    default:
      rc = ashqk_linear_workspace_size(M, N, K, G, &bytes);
  }
  check_rc(rc, "workspace_size");
  at::Tensor ws = workspace_for(x.device(), bytes);
  void* wsp = ws.defined() ? ws.data_ptr() : nullptr;
  const size_t wsb = ws.defined() ? static_cast<size_t>(ws.numel()) : 0;
  void* stream = c10::cuda::getCurrentCUDAStream(x.device().index()).stream();
  switch (path) {
    case Path::kGemv:
      rc = ashqk_w4a16_gemv(x.data_ptr(), x.stride(0), qw.data_ptr<int32_t>(), qw.stride(0),
                            qz.data_ptr<int32_t>(), qz.stride(0), s.data_ptr(), s.stride(0), y.data_ptr(),
                            y.stride(0), M, N, K, G, static_cast<int>(split_k), wsp, wsb, stream);
      break;
    case Path::kGemm:
      rc = ashqk_w4a16_gemm(x.data_ptr(), x.stride(0), qw.data_ptr<int32_t>(), qw.stride(0),
                            qz.data_ptr<int32_t>(), qz.stride(0), s.data_ptr(), s.stride(0), y.data_ptr(),
                            y.stride(0), M, N, K, G, wsp, wsb, stream);
      break;
    default:
      rc = ashqk_w4a16_linear(x.data_ptr(), x.stride(0), qw.data_ptr<int32_t>(), qw.stride(0),
                              qz.data_ptr<int32_t>(), qz.stride(0), s.data_ptr(), s.stride(0), y.data_ptr(),
                              y.stride(0), M, N, K, G, wsp, wsb, stream);
  }
  check_rc(rc, "w4a16 launch");
  return y;
}

at::Tensor w4a16_gemv(const at::Tensor& x, const at::Tensor& qw, const at::Tensor& qz, const at::Tensor& s,
                      int64_t split_k) {
  return run_linear(Path::kGemv, x, qw, qz, s, split_k, c10::nullopt);
}

at::Tensor w4a16_gemm(const at::Tensor& x, const at::Tensor& qw, const at::Tensor& qz, const at::Tensor& s) {
  return run_linear(Path::kGemm, x, qw, qz, s, 0, c10::nullopt);
}

at::Tensor w4a16_linear(const at::Tensor& x, const at::Tensor& qw, const at::Tensor& qz, const at::Tensor& s) {
  return run_linear(Path::kLinear, x, qw, qz, s, 0, c10::nullopt);
}

at::Tensor w4a16_linear_out(const at::Tensor& x, const at::Tensor& qw, const at::Tensor& qz, const at::Tensor& s,
                            at::Tensor out) {
  run_linear(Path::kLinear, x, qw, qz, s, 0, out);
  return out;
}

at::Tensor dequantize_awq(const at::Tensor& qw_in, const at::Tensor& qz_in, const at::Tensor& s_in,
                          at::ScalarType dtype) {
  TORCH_CHECK(qw_in.is_cuda(), "ashqk: qweight must be a CUDA tensor");
  TORCH_CHECK(qw_in.scalar_type() == at::kInt && qw_in.dim() == 2, "ashqk: qweight must be a 2-D int32 tensor");
  TORCH_CHECK(qz_in.scalar_type() == at::kInt && qz_in.dim() == 2, "ashqk: qzeros must be a 2-D int32 tensor");
  TORCH_CHECK(s_in.scalar_type() == at::kHalf && s_in.dim() == 2, "ashqk: scales must be a 2-D float16 tensor");
  TORCH_CHECK(dtype == at::kHalf || dtype == at::kFloat, "ashqk: dequantize_awq supports float16 and float32");
  TORCH_CHECK(qz_in.device() == qw_in.device() && s_in.device() == qw_in.device(),
              "ashqk: all tensors must be on the same device");
  c10::cuda::CUDAGuard guard(qw_in.device());
  at::Tensor qw = unit_inner(qw_in), qz = unit_inner(qz_in), s = unit_inner(s_in);
  const int64_t K = qw.size(0), N = qw.size(1) * 8;
  TORCH_CHECK(s.size(0) > 0 && K % s.size(0) == 0, "ashqk: K must be a multiple of scales.shape[0]");
  const int64_t G = K / s.size(0);
  TORCH_CHECK(qz.size(0) == K / G && qz.size(1) == N / 8 && s.size(1) == N, "ashqk: inconsistent AWQ shapes");
  at::Tensor w = at::empty({K, N}, qw.options().dtype(dtype));
  if (K == 0 || N == 0) return w;
  void* stream = c10::cuda::getCurrentCUDAStream(qw.device().index()).stream();
  int rc;
  if (dtype == at::kHalf) {
    rc = ashqk_dequantize_awq_f16(qw.data_ptr<int32_t>(), qw.stride(0), qz.data_ptr<int32_t>(), qz.stride(0),
                                  s.data_ptr(), s.stride(0), w.data_ptr(), w.stride(0), static_cast<int>(N),
                                  static_cast<int>(K), static_cast<int>(G), stream);
  } else {
    rc = ashqk_dequantize_awq_f32(qw.data_ptr<int32_t>(), qw.stride(0), qz.data_ptr<int32_t>(), qz.stride(0),
                                  s.data_ptr(), s.stride(0), w.data_ptr<float>(), w.stride(0), static_cast<int>(N),
                                  static_cast<int>(K), static_cast<int>(G), stream);
  }
  check_rc(rc, "dequantize_awq");
  return w;
}

// ---- microscaled 4-bit floating point ----------------------------------------------------------

int fp4_dtype(at::ScalarType t) {
  return t == at::kHalf ? ASHQK_F16 : t == at::kBFloat16 ? ASHQK_BF16 : t == at::kFloat ? ASHQK_F32 : -1;
}

// A tensor with rows of `cols` values as a matrix the kernels take: unit column stride, rows that do not
// overlap. A copy only where the caller's layout is neither.
struct Rows {
  at::Tensor t;
  int64_t rows, ld;
};

Rows as_rows(const at::Tensor& x, int64_t cols) {
  Rows r;
  r.t = x.dim() == 2 ? x : x.reshape({cols ? x.numel() / cols : 0, cols});
  if (r.t.stride(1) != 1 || (r.t.size(0) > 1 && r.t.stride(0) < cols)) r.t = r.t.contiguous();
  r.rows = r.t.size(0);
  r.ld = r.rows > 1 ? r.t.stride(0) : (cols + 31) / 32 * 32;  // of one row only its start's alignment counts
  TORCH_CHECK(r.rows <= INT32_MAX, "ashqk: problem too large");
  return r;
}

void check_no_grad(const at::Tensor& x, const char* what) {
  TORCH_CHECK(!(at::GradMode::is_enabled() && x.requires_grad()), "ashqk.", what,
              " has no gradient: call it under torch.no_grad() or with x.detach()");
}

void check_fp4(const at::Tensor& codes, const at::Tensor& scales, int64_t K, int64_t format, const at::Device& dev) {
  TORCH_CHECK(K > 0 && K <= (1 << 24), "ashqk: K out of range");
  TORCH_CHECK(codes.device() == dev && scales.device() == dev, "ashqk: all tensors must be on the same device");
  TORCH_CHECK(codes.scalar_type() == at::kByte && codes.dim() == 2 && codes.size(1) == (K + 31) / 32 * 16 &&
                  codes.stride(1) == 1,
              "ashqk: codes must be uint8 [rows, ceil(K / 32) * 16] with unit column stride");
  TORCH_CHECK(codes.size(0) <= INT32_MAX, "ashqk: problem too large");
  int64_t ld = 0, bytes = 0;
  TORCH_CHECK(ashqk_fp4_sizes(static_cast<int>(codes.size(0)), static_cast<int>(K), static_cast<int>(format), &ld, &bytes) == ASHQK_OK,
              "ashqk: unknown 4-bit format ", format);
  TORCH_CHECK(scales.scalar_type() == at::kByte && scales.is_contiguous() && scales.numel() == bytes,
              "ashqk: scales must be contiguous uint8 [ceil(rows / 128), ceil(blocks / 4), 32, 4, 4]");
}

int64_t codes_ld(const at::Tensor& codes) { return codes.size(0) > 1 ? codes.stride(0) : codes.size(1); }

// A new tensor straight from the CUDA allocator: at::empty comes to the same place by way of the dispatcher (a call
// that makes two tensors: 7.1 us of host time instead of 6.7).
at::Tensor new_cuda(at::IntArrayRef shape, at::ScalarType dtype, const at::Device& dev) {
  return at::Tensor(at::detail::empty_cuda(shape, dtype, dev, c10::nullopt));
}

at::Tensor empty_scales(int64_t rows, int64_t K, int64_t format, const at::Device& dev) {
  const int64_t blocks = (K + 31) / 32 * (format == ASHQK_MXFP4 ? 1 : 2);
  return new_cuda({(rows + 127) / 128, (blocks + 3) / 4, 32, 4, 4}, at::kByte, dev);
}

std::tuple<at::Tensor, at::Tensor> quantize_fp4(const at::Tensor& x, int64_t format, double global_scale, bool gated) {
  TORCH_CHECK(x.is_cuda(), "ashqk: x must be a CUDA tensor");
  const int dtype = fp4_dtype(x.scalar_type());
  TORCH_CHECK(dtype >= 0 && x.dim() >= 1, "ashqk: x must be a float16, bfloat16 or float32 tensor of at least one dimension");
  check_no_grad(x, "quantize_fp4");
  TORCH_CHECK(format == ASHQK_MXFP4 || format == ASHQK_NVFP4, "ashqk: unknown 4-bit format ", format);
  const int64_t cols = x.size(-1), K = gated ? cols / 2 : cols;
  TORCH_CHECK(K > 0 && K <= (1 << 24) && (!gated || cols % 2 == 0), "ashqk: x needs columns (an even number when gated)");
  c10::cuda::CUDAGuard guard(x.device());
  const Rows r = as_rows(x, cols);
  at::Tensor codes = new_cuda({r.rows, (K + 31) / 32 * 16}, at::kByte, x.device());
  at::Tensor scales = empty_scales(r.rows, K, format, x.device());
  if (r.rows == 0) return {codes, scales};
  check_rc(ashqk_quantize_fp4(r.t.data_ptr(), r.ld, dtype, gated, codes.data_ptr(), codes.size(1), scales.data_ptr(),
                              static_cast<int>(r.rows), static_cast<int>(K), static_cast<int>(format),
                              static_cast<float>(global_scale), c10::cuda::getCurrentCUDAStream(x.device().index()).stream()),
           "quantize_fp4");
  return {codes, scales};
}

at::Tensor dequantize_fp4(const at::Tensor& codes, const at::Tensor& scales, int64_t K, int64_t format,
                          double global_scale, at::ScalarType dtype) {
  TORCH_CHECK(codes.is_cuda(), "ashqk: codes must be a CUDA tensor");
  TORCH_CHECK(fp4_dtype(dtype) >= 0, "ashqk: dequantize_fp4 supports float16, bfloat16 and float32");
  check_fp4(codes, scales, K, format, codes.device());
  c10::cuda::CUDAGuard guard(codes.device());
  at::Tensor out = new_cuda({codes.size(0), K}, dtype, codes.device());
  if (codes.size(0) == 0) return out;
  check_rc(ashqk_dequantize_fp4(codes.data_ptr(), codes_ld(codes), scales.data_ptr(), out.data_ptr(), K, fp4_dtype(dtype),
                                static_cast<int>(codes.size(0)), static_cast<int>(K), static_cast<int>(format),
                                static_cast<float>(global_scale),
                                c10::cuda::getCurrentCUDAStream(codes.device().index()).stream()),
           "dequantize_fp4");
  return out;
}

at::Tensor fp4_matmul(const at::Tensor& a_codes, const at::Tensor& a_scales, const at::Tensor& b_codes,
                      const at::Tensor& b_scales, int64_t K, int64_t format, double alpha, at::ScalarType dtype) {
  TORCH_CHECK(a_codes.is_cuda(), "ashqk: codes must be CUDA tensors");
  TORCH_CHECK(dtype == at::kHalf || dtype == at::kBFloat16, "ashqk: fp4_matmul returns float16 or bfloat16");
  check_fp4(a_codes, a_scales, K, format, a_codes.device());
  check_fp4(b_codes, b_scales, K, format, a_codes.device());
  c10::cuda::CUDAGuard guard(a_codes.device());
  const int64_t M = a_codes.size(0), N = b_codes.size(0);
  at::Tensor y = new_cuda({M, N}, dtype, a_codes.device());
  if (M == 0 || N == 0) return y;
  check_rc(ashqk_fp4_matmul(a_codes.data_ptr(), codes_ld(a_codes), a_scales.data_ptr(), b_codes.data_ptr(),
                            codes_ld(b_codes), b_scales.data_ptr(), y.data_ptr(), N, fp4_dtype(dtype), static_cast<int>(M),
                            static_cast<int>(N), static_cast<int>(K), static_cast<int>(format), static_cast<float>(alpha),
                            c10::cuda::getCurrentCUDAStream(a_codes.device().index()).stream()),
           "fp4_matmul");
  return y;
}

at::Tensor w4a4_linear(const at::Tensor& x, const at::Tensor& codes, const at::Tensor& scales, int64_t K,
                       int64_t format, double x_scale, double w_scale, bool gated) {
  TORCH_CHECK(x.is_cuda(), "ashqk: x must be a CUDA tensor");
  const int dtype = fp4_dtype(x.scalar_type());
  TORCH_CHECK((dtype == ASHQK_F16 || dtype == ASHQK_BF16) && x.dim() >= 1, "ashqk: x must be a float16 or bfloat16 tensor");
  check_no_grad(x, "w4a4_linear");
  const int64_t cols = gated ? 2 * K : K;
  TORCH_CHECK(x.size(-1) == cols, "ashqk: x must have ", cols, " columns for weights of K = ", K, gated ? " (gated)" : "");
  check_fp4(codes, scales, K, format, x.device());
  c10::cuda::CUDAGuard guard(x.device());
  const Rows r = as_rows(x, cols);
  const int64_t N = codes.size(0);
  at::Tensor y = new_cuda({r.rows, N}, x.scalar_type(), x.device());
  if (r.rows > 0 && N > 0) {
    size_t bytes = 0;
    check_rc(ashqk_w4a4_workspace_size(static_cast<int>(r.rows), static_cast<int>(N), static_cast<int>(K), static_cast<int>(format), gated, &bytes), "w4a4_linear");
    // Holds x quantised between two launches; from PyTorch's allocator, so streams and graphs each have their own.
    at::Tensor ws;
    if (bytes) ws = new_cuda({static_cast<int64_t>(bytes)}, at::kByte, x.device());
    check_rc(ashqk_w4a4_linear(r.t.data_ptr(), r.ld, dtype, gated, static_cast<float>(x_scale), codes.data_ptr(), codes_ld(codes),
                               scales.data_ptr(), static_cast<float>(w_scale), y.data_ptr(), N, static_cast<int>(r.rows),
                               static_cast<int>(N), static_cast<int>(K), static_cast<int>(format),
                               bytes ? ws.data_ptr() : nullptr, bytes,
                               c10::cuda::getCurrentCUDAStream(x.device().index()).stream()),
             "w4a4_linear");
  }
  if (x.dim() == 2) return y;
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = N;
  return y.view(shape);
}

}  // namespace

TORCH_LIBRARY(ashqk, m) {
  m.def("w4a16_gemv(Tensor x, Tensor qweight, Tensor qzeros, Tensor scales, int split_k=0) -> Tensor");
  m.def("w4a16_gemm(Tensor x, Tensor qweight, Tensor qzeros, Tensor scales) -> Tensor");
  m.def("w4a16_linear(Tensor x, Tensor qweight, Tensor qzeros, Tensor scales) -> Tensor");
  m.def("w4a16_linear_out(Tensor x, Tensor qweight, Tensor qzeros, Tensor scales, Tensor(a!) out) -> Tensor(a!)");
  m.def("dequantize_awq(Tensor qweight, Tensor qzeros, Tensor scales, ScalarType dtype) -> Tensor");
  m.def("quantize_fp4(Tensor x, int format, float global_scale, bool gated) -> (Tensor, Tensor)");
  m.def("dequantize_fp4(Tensor codes, Tensor scales, int K, int format, float global_scale, ScalarType dtype) -> Tensor");
  m.def(
      "fp4_matmul(Tensor a_codes, Tensor a_scales, Tensor b_codes, Tensor b_scales, int K, int format, float alpha, "
      "ScalarType dtype) -> Tensor");
  m.def(
      "w4a4_linear(Tensor x, Tensor codes, Tensor scales, int K, int format, float x_scale, float w_scale, bool gated) "
      "-> Tensor");
}

TORCH_LIBRARY_IMPL(ashqk, CUDA, m) {
  m.impl("w4a16_gemv", &w4a16_gemv);
  m.impl("w4a16_gemm", &w4a16_gemm);
  m.impl("w4a16_linear", &w4a16_linear);
  m.impl("w4a16_linear_out", &w4a16_linear_out);
  m.impl("dequantize_awq", &dequantize_awq);
  m.impl("quantize_fp4", &quantize_fp4);
  m.impl("dequantize_fp4", &dequantize_fp4);
  m.impl("fp4_matmul", &fp4_matmul);
  m.impl("w4a4_linear", &w4a4_linear);
}
