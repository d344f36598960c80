// Quantising rows to microscaled 4-bit floating point, plain or of silu(gate) * up, and reading
// them back.
//
// One thread takes chunks of sixteen columns (one 32-byte load of a 16-bit input, 8 bytes of codes): an NVFP4 block, or
// half an MXFP4 block, whose two lanes share its largest magnitude by a shuffle. Every value is read once and
// nothing passes through shared memory. A value costs its input, half a byte of code and 1/32 or 1/16
// byte of scale; the arithmetic is in pairs (f32x2) because at HBM speed an SM has some eleven instruction slots
// per value. Where there are enough chunks a thread takes two, their loads in flight together.
#include <algorithm>

#include "fp4.cuh"
#include "sm100.cuh"

namespace ashqk {
namespace {

constexpr int kQuantThreads = 256;

// i / d for i < 2^31 by a multiplication: m = ceil(2^(31 + s) / d) with 2^(s-1) < d <= 2^s has an error small enough
// for 31-bit numerators (T. Granlund, P. L. Montgomery, Division by invariant integers using
// multiplication, 1994).
struct FastDiv {
  uint32_t d, mul, shift;
};
FastDiv fast_div(uint32_t d) {
  uint32_t s = 0;
  while ((1ull << s) < d) ++s;
  return {d, static_cast<uint32_t>(((1ull << (31 + s)) + d - 1) / d), s};
}
__device__ __forceinline__ uint32_t divide(uint32_t i, const FastDiv& f) {
  return static_cast<uint32_t>((static_cast<uint64_t>(i) * f.mul) >> (31 + f.shift));
}

// WHOLE: every row is whole tiles of four blocks, whose scales then leave as one 4-byte store.
template <int FMT, typename T, bool GATED, int BATCH, bool WHOLE>
__global__ void __launch_bounds__(kQuantThreads)
    quantize_fp4_kernel(const T* x, int64_t x_ld, uint8_t* __restrict__ codes, int64_t codes_ld,
                        uint8_t* __restrict__ scales, int64_t row0, uint32_t total, int K, FastDiv by_chunks, Fp4Quant q,
                        int align, int early) {
  constexpr int kLanes = fp4_block(FMT) / 16;  // lanes of a block
  pdl_wait();
  if (early) pdl_launch_dependents();
  const uint32_t chunks = by_chunks.d;  // of a row; an even number: a block's lanes share a row
  const int64_t tiles = fp4_scale_tiles(K, FMT);
  const uint32_t first = blockIdx.x * (kQuantThreads * BATCH) + threadIdx.x;
  Raw16<T> g[BATCH], u[GATED ? BATCH : 1];
  uint32_t row[BATCH], chunk[BATCH];
#pragma unroll
  for (int b = 0; b < BATCH; ++b) {
    const uint32_t i = first + b * kQuantThreads;
    row[b] = divide(i, by_chunks);
    chunk[b] = i - row[b] * chunks;
    const int k0 = static_cast<int>(chunk[b]) * 16;
#pragma unroll
    for (int j = 0; j < static_cast<int>(4 * sizeof(T)); ++j) {
      g[b].w[j] = 0;
      if (GATED) u[b].w[j] = 0;
    }
    if (i < total && k0 < K) {
      const T* p = x + (row0 + row[b]) * x_ld + k0;
      const int al = k0 + 16 <= K ? align : 0;
      load16<T>(p, K - k0, al, g[b]);
      if (GATED) load16<T>(p + K, K - k0, al, u[b]);
    }
  }
#pragma unroll
  for (int b = 0; b < BATCH; ++b) {
    float v[16];
    unpack16<T>(g[b], v);
    uint32_t amax;
    if constexpr (GATED) {
      float w[16];
      unpack16<T>(u[b], w);
#pragma unroll
      for (int j = 0; j < 16; ++j) v[j] = silu_mul(v[j], w[j]);
      amax = abs_max16(v);
    } else {
      amax = abs_max16(g[b]);
    }
    uint2 c;
    uint32_t bytes = fp4_quantize16<FMT>(v, amax, q, &c);
    const int block = static_cast<int>(chunk[b] / kLanes);
    if (WHOLE) {
      bytes <<= 8 * (block & 3);
      bytes |= __shfl_xor_sync(0xffffffffu, bytes, kLanes);
      bytes |= __shfl_xor_sync(0xffffffffu, bytes, 2 * kLanes);
    }
    if (first + b * kQuantThreads >= total) continue;
    const int64_t r = row0 + row[b];
    *reinterpret_cast<uint2*>(codes + r * codes_ld + chunk[b] * 8) = c;
    uint8_t* s = scales + fp4_scale_offset(r, block, tiles);
    if (WHOLE) {
      if (chunk[b] % (4 * kLanes) == 0) *reinterpret_cast<uint32_t*>(s) = bytes;
    } else if (chunk[b] % kLanes == 0) {
      *s = static_cast<uint8_t>(bytes);
      if (chunk[b] + kLanes == chunks)  // the tile's padding blocks
        for (int k = block + 1; k & 3; ++k) *++s = 0;
    }
  }
}

template <int FMT, typename T, int BATCH>
__global__ void __launch_bounds__(kQuantThreads)
    dequantize_fp4_kernel(const uint8_t* codes, int64_t codes_ld, const uint8_t* scales, T* __restrict__ out,
                          int64_t out_ld, int64_t row0, uint32_t total, int K, FastDiv by_chunks, float gs, bool vec) {
  pdl_wait();
  const uint32_t chunks = by_chunks.d;
  const int64_t tiles = fp4_scale_tiles(K, FMT);
  const uint32_t first = blockIdx.x * (kQuantThreads * BATCH) + threadIdx.x;
  uint32_t c[BATCH], s[BATCH];
#pragma unroll
  for (int b = 0; b < BATCH; ++b) {
    const uint32_t i = first + b * kQuantThreads;
    const uint32_t r = divide(i, by_chunks);
    const uint32_t chunk = i - r * chunks;
    c[b] = s[b] = 0;
    if (i < total) {
      c[b] = *reinterpret_cast<const uint32_t*>(codes + (row0 + r) * codes_ld + chunk * 4);
      s[b] = scales[fp4_scale_offset(row0 + r, static_cast<int>(chunk * 8 / fp4_block(FMT)), tiles)];
    }
  }
#pragma unroll
  for (int b = 0; b < BATCH; ++b) {
    const uint32_t i = first + b * kQuantThreads;
    if (i >= total) break;
    const uint32_t r = divide(i, by_chunks);
    const int k0 = static_cast<int>(i - r * chunks) * 8;
    float v[8];
    fp4_unpack8(c[b], v);
    const float sv = fp4_scale_value<FMT>(s[b]);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = v[j] * sv * gs;
    T* o = out + (row0 + r) * out_ld + k0;
    if (vec && k0 + 8 <= K) {
      if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<uint4*>(o) =
            make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
      } else {
        reinterpret_cast<float4*>(o)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(o)[1] = make_float4(v[4], v[5], v[6], v[7]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (k0 + j < K) o[j] = from_f32<T>(v[j]);
    }
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

constexpr int kQuantBatch = 2, kDequantBatch = 4;
// Whether `batch` chunks per thread still leave every SM two blocks (148 SMs).
constexpr bool many_chunks(int64_t chunks, int batch) { return chunks >= 2 * 148 * kQuantThreads * batch; }

// Calls launch(row0, chunks, blocks of kQuantThreads * batch) for slabs of rows with fewer than 2^31 chunks.
template <typename F>
int for_slabs(int64_t rows, int64_t chunks, int batch, F launch) {
  const int64_t most = std::max<int64_t>(1, ((1ll << 31) - 8 * kQuantThreads) / chunks);
  for (int64_t row0 = 0; row0 < rows; row0 += most) {
    const int64_t total = std::min(most, rows - row0) * chunks;
    if (const int rc = launch(row0, static_cast<uint32_t>(total), ceil_div64(total, kQuantThreads * batch))) return rc;
  }
  return ASHQK_OK;
}

template <int FMT, typename T, bool GATED, int BATCH, bool WHOLE>
int quantize_launch(const void* x, int64_t x_ld, uint8_t* codes, int64_t codes_ld, uint8_t* scales, int M, int K, float gs,
                    bool early, cudaStream_t stream) {
  int align = chunk_align(x, x_ld, sizeof(T));
  if (GATED) align = std::min(align, chunk_align(nullptr, K, sizeof(T)));
  const int64_t chunks = fp4_padded_k(K) / 16;
  return for_slabs(M, chunks, BATCH, [&](int64_t row0, uint32_t total, int64_t blocks) {
    return launch_pdl(quantize_fp4_kernel<FMT, T, GATED, BATCH, WHOLE>, blocks, kQuantThreads, stream,
                      static_cast<const T*>(x), x_ld, codes, codes_ld, scales, row0, total, K,
                      fast_div(static_cast<uint32_t>(chunks)), fp4_quant_params(gs), align, early);
  });
}

template <int FMT, typename T, bool GATED>
int quantize_shaped(const void* x, int64_t x_ld, uint8_t* codes, int64_t codes_ld, uint8_t* scales, int M, int K, float gs,
                    bool early, cudaStream_t stream) {
  const int64_t kp = fp4_padded_k(K);
  const bool whole = kp % (4 * fp4_block(FMT)) == 0;
  const bool many = many_chunks(M * (kp / 16), kQuantBatch);
  return (whole ? many ? quantize_launch<FMT, T, GATED, kQuantBatch, true> : quantize_launch<FMT, T, GATED, 1, true>
          : many ? quantize_launch<FMT, T, GATED, kQuantBatch, false>
                 : quantize_launch<FMT, T, GATED, 1, false>)(x, x_ld, codes, codes_ld, scales, M, K, gs, early, stream);
}

template <int FMT, typename T>
int quantize_typed(const void* x, int64_t x_ld, bool gated, uint8_t* codes, int64_t codes_ld, uint8_t* scales, int M,
                   int K, float gs, bool early, cudaStream_t stream) {
  return gated ? quantize_shaped<FMT, T, true>(x, x_ld, codes, codes_ld, scales, M, K, gs, early, stream)
               : quantize_shaped<FMT, T, false>(x, x_ld, codes, codes_ld, scales, M, K, gs, early, stream);
}

template <int FMT, typename T>
int dequantize_typed(const uint8_t* codes, int64_t codes_ld, const uint8_t* scales, void* out, int64_t out_ld, int M,
                     int K, float gs, cudaStream_t stream) {
  const bool vec = aligned(out, 16) && (out_ld * sizeof(T)) % 16 == 0;
  const int64_t chunks = (K + 7) / 8;
  const bool many = many_chunks(M * chunks, kDequantBatch);
  return for_slabs(M, chunks, many ? kDequantBatch : 1, [&](int64_t row0, uint32_t total, int64_t blocks) {
    return launch_pdl(many ? dequantize_fp4_kernel<FMT, T, kDequantBatch> : dequantize_fp4_kernel<FMT, T, 1>, blocks,
                      kQuantThreads, stream, codes, codes_ld, scales, static_cast<T*>(out), out_ld, row0, total, K,
                      fast_div(static_cast<uint32_t>(chunks)), gs, vec);
  });
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
