// Quantising rows to microscaled 4-bit floating point, plain or of silu(gate) * up, and reading
// them back.
//
// One thread takes eight columns (16 bytes of a 16-bit input, 4 bytes of codes); the lanes of a block
// (4 for MXFP4, 2 for NVFP4) share its largest magnitude by shuffles, so every value is read once and
// nothing passes through shared memory. HBM-bound: a value costs its input, half a byte of code and
// 1/32 or 1/16 byte of scale.
#include <type_traits>

#include "fp4.cuh"
#include "sm100.cuh"

namespace ashqk {
namespace {

constexpr int kQuantThreads = 256;

template <int FMT, typename T, bool GATED>
__global__ void __launch_bounds__(kQuantThreads)
    quantize_fp4_kernel(const T* x, int64_t x_ld, uint8_t* __restrict__ codes, int64_t codes_ld,
                        uint8_t* __restrict__ scales, int64_t rows, int K, float gs, bool vec, int early) {
  constexpr int kLanes = fp4_block(FMT) / 8;  // lanes of a block
  pdl_wait();
  if (early) pdl_launch_dependents();
  const int chunks = static_cast<int>(fp4_padded_k(K) / 8);  // a multiple of 4: a block's lanes share a row
  const int64_t tiles = fp4_scale_tiles(K, FMT);
  const int64_t idx = static_cast<int64_t>(blockIdx.x) * kQuantThreads + threadIdx.x;
  const bool live = idx < rows * chunks;
  const int64_t row = live ? idx / chunks : 0;
  const int chunk = live ? static_cast<int>(idx - row * chunks) : 0;
  const int k0 = chunk * 8;
  float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (live && k0 < K) {
    const T* p = x + row * x_ld + k0;
    const bool whole = vec && k0 + 8 <= K;
    load8<T>(p, K - k0, whole, v);
    if (GATED) {
      float u[8];
      load8<T>(p + K, K - k0, whole, u);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = silu_mul(v[i], u[i]);
    }
  }
  uint32_t amax = abs_max8(v);
#pragma unroll
  for (int d = 1; d < kLanes; d *= 2) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, d));
  if (!live) return;
  float divisor;
  const uint32_t byte = fp4_scale_of<FMT>(amax, gs, &divisor);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = fp4_scaled<FMT>(v[i], divisor);
  *reinterpret_cast<uint32_t*>(codes + row * codes_ld + chunk * 4) = fp4_pack8(v);
  if (chunk % kLanes == 0) {
    const int block = chunk / kLanes;
    uint8_t* s = scales + fp4_scale_offset(row, block, tiles);
    *s = static_cast<uint8_t>(byte);
    if (block == chunks / kLanes - 1)  // the tile's padding blocks
      for (int b = block + 1; b & 3; ++b) *++s = 0;
  }
}

template <int FMT, typename T>
__global__ void __launch_bounds__(kQuantThreads)
    dequantize_fp4_kernel(const uint8_t* codes, int64_t codes_ld, const uint8_t* scales,
                          T* __restrict__ out, int64_t out_ld, int64_t rows, int K, float gs, bool vec) {
  pdl_wait();
  const int chunks = (K + 7) / 8;
  const int64_t tiles = fp4_scale_tiles(K, FMT);
  const int64_t idx = static_cast<int64_t>(blockIdx.x) * kQuantThreads + threadIdx.x;
  if (idx >= rows * chunks) return;
  const int64_t row = idx / chunks;
  const int chunk = static_cast<int>(idx - row * chunks);
  const int k0 = chunk * 8;
  float v[8];
  fp4_unpack8(*reinterpret_cast<const uint32_t*>(codes + row * codes_ld + chunk * 4), v);
  const float s = fp4_scale_value<FMT>(scales[fp4_scale_offset(row, k0 / fp4_block(FMT), tiles)]);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = v[i] * s * gs;
  T* o = out + row * out_ld + k0;
  if (vec && k0 + 8 <= K) {
    if (sizeof(T) == 2) {
      using H = std::conditional_t<sizeof(T) == 2, T, __half>;
      *reinterpret_cast<uint4*>(o) =
          make_uint4(pack2<H>(v[0], v[1]), pack2<H>(v[2], v[3]), pack2<H>(v[4], v[5]), pack2<H>(v[6], v[7]));
    } else {
      reinterpret_cast<float4*>(o)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(o)[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (k0 + i < K) o[i] = from_f32<T>(v[i]);
  }
}

template <typename... Params, typename... Args>
int launch_pdl(void (*kernel)(Params...), int64_t blocks, int threads, cudaStream_t stream, Args... args) {
  if (blocks > 0x7fffffff) return ASHQK_ERR_UNSUPPORTED;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = pdl_enabled() ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...) == cudaSuccess ? ASHQK_OK : ASHQK_ERR_CUDA;
}

template <int FMT, typename T>
int quantize_typed(const void* x, int64_t x_ld, bool gated, uint8_t* codes, int64_t codes_ld, uint8_t* scales, int M,
                   int K, float gs, bool early, cudaStream_t stream) {
  const bool vec = aligned(x, 16) && (x_ld * sizeof(T)) % 16 == 0 && (!gated || (K * sizeof(T)) % 16 == 0);
  const int64_t blocks = ceil_div64(M * (fp4_padded_k(K) / 8), kQuantThreads);
  const T* xt = static_cast<const T*>(x);
  return gated ? launch_pdl(quantize_fp4_kernel<FMT, T, true>, blocks, kQuantThreads, stream, xt, x_ld, codes,
                            codes_ld, scales, M, K, gs, vec, early)
               : launch_pdl(quantize_fp4_kernel<FMT, T, false>, blocks, kQuantThreads, stream, xt, x_ld, codes,
                            codes_ld, scales, M, K, gs, vec, early);
}

template <int FMT, typename T>
int dequantize_typed(const uint8_t* codes, int64_t codes_ld, const uint8_t* scales, void* out, int64_t out_ld, int M,
                     int K, float gs, cudaStream_t stream) {
  const bool vec = aligned(out, 16) && (out_ld * sizeof(T)) % 16 == 0;
  const int64_t blocks = ceil_div64(static_cast<int64_t>(M) * ((K + 7) / 8), kQuantThreads);
  return launch_pdl(dequantize_fp4_kernel<FMT, T>, blocks, kQuantThreads, stream, codes, codes_ld, scales,
                    static_cast<T*>(out), out_ld, M, K, gs, vec);
}

}  // namespace

int dtype_size(int dtype) { return dtype == ASHQK_F32 ? 4 : (dtype == ASHQK_F16 || dtype == ASHQK_BF16) ? 2 : 0; }

int check_fp4_operand(const void* codes, int64_t codes_ld, const void* scales, int K) {
  if (!codes || !scales || !aligned(codes, 16) || !aligned(scales, 16)) return ASHQK_ERR_INVALID_ARGUMENT;
  if (codes_ld % 16 || codes_ld < fp4_padded_k(K) / 2) return ASHQK_ERR_INVALID_ARGUMENT;
  return ASHQK_OK;
}

bool fp4_global_scale_ok(int format, float gs) {
  return format == ASHQK_MXFP4 ? gs == 1.0f : gs >= 1e-18f && gs <= 1e18f;
}

// `early`: let the next launch start while this one runs. Only for a consumer that reads the result
// behind its own griddepcontrol.wait, which a product reading these codes as weights does not.
int quantize_fp4(const void* x, int64_t x_ld, int dtype, bool gated, void* codes, int64_t codes_ld, void* scales, int M,
                 int K, int format, float gs, bool early, cudaStream_t stream) {
  uint8_t* c = static_cast<uint8_t*>(codes);
  uint8_t* s = static_cast<uint8_t*>(scales);
#define ASHQK_QUANT(FMT, T) quantize_typed<FMT, T>(x, x_ld, gated, c, codes_ld, s, M, K, gs, early, stream)
  if (format == ASHQK_MXFP4)
    return dtype == ASHQK_F16    ? ASHQK_QUANT(ASHQK_MXFP4, __half)
           : dtype == ASHQK_BF16 ? ASHQK_QUANT(ASHQK_MXFP4, __nv_bfloat16)
                                 : ASHQK_QUANT(ASHQK_MXFP4, float);
  return dtype == ASHQK_F16    ? ASHQK_QUANT(ASHQK_NVFP4, __half)
         : dtype == ASHQK_BF16 ? ASHQK_QUANT(ASHQK_NVFP4, __nv_bfloat16)
                               : ASHQK_QUANT(ASHQK_NVFP4, float);
#undef ASHQK_QUANT
}

}  // namespace ashqk

using namespace ashqk;

extern "C" int ashqk_fp4_sizes(int M, int K, int format, int64_t* codes_ld, int64_t* scales_bytes) {
  if (M < 0 || K <= 0 || !fp4_format_ok(format) || !codes_ld || !scales_bytes) return ASHQK_ERR_INVALID_ARGUMENT;
  *codes_ld = fp4_padded_k(K) / 2;
  *scales_bytes = ceil_div64(M, kFp4TileRows) * fp4_scale_tiles(K, format) * kFp4TileBytes;
  return ASHQK_OK;
}

extern "C" int ashqk_quantize_fp4(const void* x, int64_t x_ld, int dtype, int gated, void* codes, int64_t codes_ld,
                                  void* scales, int M, int K, int format, float global_scale, void* stream) {
  const int size = dtype_size(dtype);
  if (!x || M <= 0 || K <= 0 || K > (1 << 30) || !size || !aligned(x, size) || !fp4_format_ok(format)) return ASHQK_ERR_INVALID_ARGUMENT;
  if (x_ld < static_cast<int64_t>(K) * (gated ? 2 : 1) || !fp4_global_scale_ok(format, global_scale))
    return ASHQK_ERR_INVALID_ARGUMENT;
  if (const int rc = check_fp4_operand(codes, codes_ld, scales, K)) return rc;
  return quantize_fp4(x, x_ld, dtype, gated != 0, codes, codes_ld, scales, M, K, format, global_scale, false,
                      static_cast<cudaStream_t>(stream));
}

extern "C" int ashqk_dequantize_fp4(const void* codes, int64_t codes_ld, const void* scales, void* out, int64_t out_ld,
                                    int dtype, int M, int K, int format, float global_scale, void* stream) {
  const int size = dtype_size(dtype);
  if (!out || M <= 0 || K <= 0 || K > (1 << 30) || !size || !aligned(out, size) || !fp4_format_ok(format) || out_ld < K ||
      !fp4_global_scale_ok(format, global_scale))
    return ASHQK_ERR_INVALID_ARGUMENT;
  if (const int rc = check_fp4_operand(codes, codes_ld, scales, K)) return rc;
  const uint8_t* c = static_cast<const uint8_t*>(codes);
  const uint8_t* s = static_cast<const uint8_t*>(scales);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
#define ASHQK_DEQUANT(FMT, T) dequantize_typed<FMT, T>(c, codes_ld, s, out, out_ld, M, K, global_scale, st)
  if (format == ASHQK_MXFP4)
    return dtype == ASHQK_F16    ? ASHQK_DEQUANT(ASHQK_MXFP4, __half)
           : dtype == ASHQK_BF16 ? ASHQK_DEQUANT(ASHQK_MXFP4, __nv_bfloat16)
                                 : ASHQK_DEQUANT(ASHQK_MXFP4, float);
  return dtype == ASHQK_F16    ? ASHQK_DEQUANT(ASHQK_NVFP4, __half)
         : dtype == ASHQK_BF16 ? ASHQK_DEQUANT(ASHQK_NVFP4, __nv_bfloat16)
                               : ASHQK_DEQUANT(ASHQK_NVFP4, float);
#undef ASHQK_DEQUANT
}
