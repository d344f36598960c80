// Quantising rows to microscaled 4-bit floating point, plain or of silu(gate) * up, and reading
// them back.
//
// One thread takes 32 columns: two 32-byte loads of a 16-bit input, one 16-byte store of codes, the scales of one MXFP4
// or two NVFP4 blocks. Every value is read once and nothing passes through shared memory. A value costs its input,
// half a byte of code and 1/32 or 1/16 byte of scale. At HBM speed an SM has some eleven instruction slots per
// value, so the arithmetic is in pairs (f32x2) and offsets within a launch are 32-bit. Measured at 8192 x 12288 fp16 on
// a B200 (L2 flushed): to MXFP4 47 us (5.4 TB/s), to NVFP4 51 us (5.0), gated 82 and 86 us (5.6, 5.3), read back 43 us
// (6.0); fp32 84 and 86 us (5.4, 5.3), read back 96 and 98 (4.7); 8 columns per thread and IEEE divisions took about 2.5
// times as long for NVFP4.
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

constexpr int kChunk = 32;  // columns per thread

// The rows of one launch start at `x`, `codes` and `scales` and lie in fewer than 2^31 bytes of codes.
// WHOLE: every row is whole tiles of four blocks, whose scales then leave as one 4-byte store.
template <int FMT, typename T, bool GATED, bool WHOLE>
__global__ void __launch_bounds__(kQuantThreads, sizeof(T) == 4 ? 2 : GATED ? 3 : 4)
    quantize_fp4_kernel(const T* x, int64_t x_ld, uint8_t* __restrict__ codes, uint32_t codes_ld,
                        uint8_t* __restrict__ scales, uint32_t tiles, uint32_t total, int K, FastDiv by_chunks,
                        Fp4Quant q, int align, int early) {
  constexpr int kHalves = kChunk / 16;
  constexpr int kBlocks = kChunk / fp4_block(FMT);  // of a chunk
  pdl_wait();
  if (early) pdl_launch_dependents();
  const uint32_t i = blockIdx.x * kQuantThreads + threadIdx.x;
  const uint32_t row = divide(i, by_chunks);
  const uint32_t chunk = i - row * by_chunks.d;
  const int k0 = static_cast<int>(chunk) * kChunk;
  Raw16<T> g[kHalves], u[GATED ? kHalves : 1];
  const T* p = x + row * x_ld + k0;
#pragma unroll
  for (int h = 0; h < kHalves; ++h) {
    const int left = K - k0 - 16 * h;
    const int al = left >= 16 ? align : 0;
#pragma unroll
    for (int j = 0; j < static_cast<int>(4 * sizeof(T)); ++j) {
      g[h].w[j] = 0;
      if (GATED) u[h].w[j] = 0;
    }
    if (i < total && left > 0) {
      load16<T>(p + 16 * h, left, al, g[h]);
      if (GATED) load16<T>(p + 16 * h + K, left, al, u[h]);
    }
  }
  float v[kChunk];
  uint32_t amax[kHalves];
#pragma unroll
  for (int h = 0; h < kHalves; ++h) {
    unpack16<T>(g[h], v + 16 * h);
    if constexpr (GATED) {
      float w[16];
      unpack16<T>(u[h], w);
      silu_mul16(v + 16 * h, w);
      amax[h] = abs_max16(v + 16 * h);
    } else {
      amax[h] = abs_max16(g[h]);
    }
  }
  uint2 c[kHalves];
  uint32_t bytes;
  if (FMT == ASHQK_MXFP4) {
    float d, r;
    bytes = fp4_scale_of<FMT>(max(amax[0], amax[1]), q, &d, &r);
#pragma unroll
    for (int h = 0; h < kHalves; ++h) c[h] = fp4_codes16<FMT>(v + 16 * h, bytes, d, r);
  } else {
    bytes = 0;
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      float d, r;
      const uint32_t byte = fp4_scale_of<FMT>(amax[h], q, &d, &r);
      c[h] = fp4_codes16<FMT>(v + 16 * h, byte, d, r);
      bytes |= byte << (8 * h);
    }
  }
  const uint32_t block = chunk * kBlocks;
  if (WHOLE) {  // the lanes of a tile are neighbours
    bytes <<= 8 * (block & 3);
#pragma unroll
    for (int d = 1; d < 4 / kBlocks; d *= 2) bytes |= __shfl_xor_sync(0xffffffffu, bytes, d);
  }
  if (i >= total) return;
  *reinterpret_cast<uint4*>(codes + row * codes_ld + chunk * (kChunk / 2)) = make_uint4(c[0].x, c[0].y, c[1].x, c[1].y);
  uint8_t* s = scales + fp4_scale_offset(row, block, tiles);
  if (WHOLE) {
    if ((block & 3) == 0) *reinterpret_cast<uint32_t*>(s) = bytes;
  } else {
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) s[b] = static_cast<uint8_t>(bytes >> (8 * b));
    if (chunk + 1 == by_chunks.d)  // the tile's padding blocks
      for (int k = (block & 3) + kBlocks; k < 4; ++k) s[k - (block & 3)] = 0;
  }
}

// Rows that start on 16-byte boundaries. One thread: 32 columns, one 16-byte load of codes.
template <int FMT, typename T>
__global__ void __launch_bounds__(kQuantThreads)
    dequantize_rows_kernel(const uint8_t* codes, uint32_t codes_ld, const uint8_t* scales, T* __restrict__ out,
                           int64_t out_ld, uint32_t tiles, uint32_t total, int K, FastDiv by_chunks, float gs,
                           bool wide) {
  constexpr int kBlocks = kChunk / fp4_block(FMT);
  pdl_wait();
  const uint32_t i = blockIdx.x * kQuantThreads + threadIdx.x;
  if (i >= total) return;
  const uint32_t row = divide(i, by_chunks);
  const uint32_t chunk = i - row * by_chunks.d;
  const uint32_t block = chunk * kBlocks;
  const uint4 c4 = ld_once_v4(codes + row * codes_ld + chunk * (kChunk / 2));
  const uint8_t* s = scales + fp4_scale_offset(row, block, tiles);
  const uint32_t bytes = kBlocks == 1 ? *s : *reinterpret_cast<const uint16_t*>(s);
  const uint32_t c[4] = {c4.x, c4.y, c4.z, c4.w};
  T* y = out + row * out_ld + chunk * kChunk;
  const int left = K - static_cast<int>(chunk) * kChunk;
#pragma unroll
  for (int h = 0; h < 2; ++h) {  // sixteen columns: of one block
    const float sv = fp4_scale_value<FMT>(kBlocks == 1 ? bytes : (bytes >> (8 * h)) & 0xffu);
    float v[16];
    fp4_unpack8(c[2 * h], v);
    fp4_unpack8(c[2 * h + 1], v + 8);
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = v[j] * sv * gs;
    uint32_t w[4 * sizeof(T)];
#pragma unroll
    for (int j = 0; j < static_cast<int>(4 * sizeof(T)); ++j) {
      if constexpr (sizeof(T) == 2)
        w[j] = pack2<T>(v[2 * j], v[2 * j + 1]);
      else
        w[j] = __float_as_uint(v[j]);
    }
    T* o = y + 16 * h;
    const int n = left - 16 * h;
    if (wide && n >= 16) {
#pragma unroll
      for (int j = 0; j < static_cast<int>(4 * sizeof(T)); j += 8)
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(reinterpret_cast<uint32_t*>(o) + j),
                     "r"(w[j]), "r"(w[j + 1]), "r"(w[j + 2]), "r"(w[j + 3]), "r"(w[j + 4]), "r"(w[j + 5]), "r"(w[j + 6]),
                     "r"(w[j + 7])
                     : "memory");
    } else {
      constexpr int kPer = 16 / sizeof(T);  // values in 16 bytes
#pragma unroll
      for (int j = 0; j < 16; j += kPer) {
        const uint32_t* q = w + 4 * (j / kPer);
        if (n >= j + kPer)
          *reinterpret_cast<uint4*>(o + j) = make_uint4(q[0], q[1], q[2], q[3]);
        else
#pragma unroll
          for (int k = 0; k < kPer; ++k)
            if (j + k < n) o[j + k] = from_f32<T>(v[j + k]);
      }
    }
  }
}

// Rows of any alignment. One thread writes eight columns from a 16-byte boundary of the output on: where rows start
// `mis` values behind one, those are the last `mis` of code word c - 1 and the first of word c (eight codes, all of
// one block, each).
template <int FMT, typename T, int BATCH>
__global__ void __launch_bounds__(kQuantThreads)
    dequantize_fp4_kernel(const uint8_t* codes, int64_t codes_ld, const uint8_t* scales, T* __restrict__ out,
                          int64_t out_ld, int64_t row0, uint32_t total, int K, FastDiv by_chunks, float gs) {
  pdl_wait();
  const int words = static_cast<int>(fp4_padded_k(K) / 8);
  const int64_t tiles = fp4_scale_tiles(K, FMT);
  const uint32_t first = blockIdx.x * (kQuantThreads * BATCH) + threadIdx.x;
  uint32_t c0[BATCH], c1[BATCH], s0[BATCH], s1[BATCH];
  int mis[BATCH], word[BATCH];
  T* o[BATCH];
#pragma unroll
  for (int b = 0; b < BATCH; ++b) {
    const uint32_t i = first + b * kQuantThreads;
    const uint32_t r = divide(i, by_chunks);
    const int c = static_cast<int>(i - r * by_chunks.d);
    const int64_t row = row0 + r;
    o[b] = out + row * out_ld;
    mis[b] = static_cast<int>((reinterpret_cast<uintptr_t>(o[b]) & 15u) / sizeof(T));
    word[b] = c;
    c0[b] = c1[b] = s0[b] = s1[b] = 0;
    if (i < total) {
      const uint32_t* w = reinterpret_cast<const uint32_t*>(codes + row * codes_ld);
      if (c < words) {
        c1[b] = w[c];
        s1[b] = scales[fp4_scale_offset(row, static_cast<uint32_t>(c) * 8 / fp4_block(FMT), tiles)];
      }
      if (mis[b] && c > 0) {
        c0[b] = w[c - 1];
        s0[b] = scales[fp4_scale_offset(row, static_cast<uint32_t>(c - 1) * 8 / fp4_block(FMT), tiles)];
      }
    }
  }
#pragma unroll
  for (int b = 0; b < BATCH; ++b) {
    if (first + b * kQuantThreads >= total) break;
    const int k0 = word[b] * 8 - mis[b];
    float v[8];
    fp4_unpack8(mis[b] ? __funnelshift_r(c0[b], c1[b], 4 * (8 - mis[b])) : c1[b], v);
    const float f0 = fp4_scale_value<FMT>(s0[b]), f1 = fp4_scale_value<FMT>(s1[b]);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = v[j] * (j < mis[b] ? f0 : f1) * gs;
    T* y = o[b] + k0;
    if (k0 >= 0 && k0 + 8 <= K) {
      if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<uint4*>(y) =
            make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
      } else {
        reinterpret_cast<float4*>(y)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(y)[1] = make_float4(v[4], v[5], v[6], v[7]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (k0 + j >= 0 && k0 + j < K) y[j] = from_f32<T>(v[j]);
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

constexpr int kDequantBatch = 4;

// Calls launch(row0, rows) for slabs of whole scale tiles with at most `most` rows.
template <typename F>
int for_slabs(int64_t rows, int64_t most, F launch) {
  most = std::max<int64_t>(kFp4TileRows, most / kFp4TileRows * kFp4TileRows);
  for (int64_t row0 = 0; row0 < rows; row0 += most)
    if (const int rc = launch(row0, std::min(most, rows - row0))) return rc;
  return ASHQK_OK;
}

// Where a quantiser's result goes.
struct Fp4Target {
  uint8_t* codes;
  int64_t ld;
  uint8_t* scales;
  int M, K;
  bool early;
  cudaStream_t stream;
};

template <int FMT, typename T, bool GATED, bool WHOLE>
int quantize_launch(const Fp4Source& x, const Fp4Target& t) {
  int align = chunk_align(x.x, x.ld, sizeof(T));
  if (GATED) align = std::min(align, chunk_align(nullptr, t.K, sizeof(T)));
  const int64_t chunks = fp4_padded_k(t.K) / kChunk;
  const int64_t tiles = fp4_scale_tiles(t.K, FMT);
  return for_slabs(t.M, ((1ll << 31) - 1) / t.ld, [&](int64_t row0, int64_t rows) {
    return launch_pdl(quantize_fp4_kernel<FMT, T, GATED, WHOLE>, ceil_div64(rows * chunks, kQuantThreads),
                      kQuantThreads, t.stream, static_cast<const T*>(x.x) + row0 * x.ld, x.ld, t.codes + row0 * t.ld,
                      t.ld, t.scales + row0 / kFp4TileRows * tiles * kFp4TileBytes, tiles, rows * chunks, t.K,
                      fast_div(static_cast<uint32_t>(chunks)), fp4_quant_params(x.gs), align, t.early);
  });
}

template <int FMT, typename T>
int quantize_typed(const Fp4Source& x, const Fp4Target& t) {
  const bool whole = fp4_padded_k(t.K) % (4 * fp4_block(FMT)) == 0;
  if (x.gated) return whole ? quantize_launch<FMT, T, true, true>(x, t) : quantize_launch<FMT, T, true, false>(x, t);
  return whole ? quantize_launch<FMT, T, false, true>(x, t) : quantize_launch<FMT, T, false, false>(x, t);
}

template <int FMT>
int quantize_format(const Fp4Source& x, const Fp4Target& t) {
  return x.dtype == ASHQK_F16    ? quantize_typed<FMT, __half>(x, t)
         : x.dtype == ASHQK_BF16 ? quantize_typed<FMT, __nv_bfloat16>(x, t)
                                 : quantize_typed<FMT, float>(x, t);
}

template <int FMT, typename T>
int dequantize_typed(const uint8_t* codes, int64_t codes_ld, const uint8_t* scales, void* out, int64_t out_ld, int M,
                     int K, float gs, cudaStream_t stream) {
  if (const int align = chunk_align(out, out_ld, sizeof(T))) {
    const int64_t chunks = ceil_div64(K, kChunk);
    const int64_t tiles = fp4_scale_tiles(K, FMT);
    return for_slabs(M, ((1ll << 31) - 1) / codes_ld, [&](int64_t row0, int64_t rows) {
      return launch_pdl(dequantize_rows_kernel<FMT, T>, ceil_div64(rows * chunks, kQuantThreads), kQuantThreads, stream,
                        codes + row0 * codes_ld, codes_ld, scales + row0 / kFp4TileRows * tiles * kFp4TileBytes,
                        static_cast<T*>(out) + row0 * out_ld, out_ld, tiles, rows * chunks, K,
                        fast_div(static_cast<uint32_t>(chunks)), gs, align == 32);
    });
  }
  DeviceInfo dev;
  if (const int rc = device_info(&dev)) return rc;
  const int64_t chunks = (K + 7) / 8 + 1;  // a row that starts off a boundary may touch one more
  return for_slabs(M, ((1ll << 31) - 8 * kQuantThreads) / chunks, [&](int64_t row0, int64_t rows) {
    const int64_t total = rows * chunks;
    const bool many = total >= 2ll * dev.sm_count * kQuantThreads * kDequantBatch;  // every SM still gets two blocks
    return launch_pdl(many ? dequantize_fp4_kernel<FMT, T, kDequantBatch> : dequantize_fp4_kernel<FMT, T, 1>,
                      ceil_div64(total, kQuantThreads * (many ? kDequantBatch : 1)), kQuantThreads, stream, codes, codes_ld,
                      scales, static_cast<T*>(out), out_ld, row0, total, K, fast_div(static_cast<uint32_t>(chunks)), gs);
  });
}

}  // namespace

int dtype_size(int dtype) { return dtype == ASHQK_F32 ? 4 : (dtype == ASHQK_F16 || dtype == ASHQK_BF16) ? 2 : 0; }

int check_fp4_operand(const void* codes, int64_t codes_ld, const void* scales, int K) {
  if (!codes || !scales || !aligned(codes, 16) || !aligned(scales, 16)) return ASHQK_ERR_INVALID_ARGUMENT;
  if (codes_ld % 16 || codes_ld < fp4_padded_k(K) / 2) return ASHQK_ERR_INVALID_ARGUMENT;
  if (codes_ld > kFp4MaxLd) return ASHQK_ERR_UNSUPPORTED;
  return ASHQK_OK;
}

bool fp4_global_scale_ok(int format, float gs) {
  return format == ASHQK_MXFP4 ? gs == 1.0f : gs >= 1e-18f && gs <= 1e18f;
}

int quantize_fp4(const Fp4Source& x, uint8_t* codes, int64_t codes_ld, uint8_t* scales, int M, int K, int format, bool early,
                 cudaStream_t stream) {
  const Fp4Target t = {codes, codes_ld, scales, M, K, early, stream};
  return format == ASHQK_MXFP4 ? quantize_format<ASHQK_MXFP4>(x, t) : quantize_format<ASHQK_NVFP4>(x, t);
}

}  // namespace ashqk

using namespace ashqk;

extern "C" int ashqk_fp4_sizes(int M, int K, int format, int64_t* codes_ld, int64_t* scales_bytes) {
  if (M < 0 || K <= 0 || K > kFp4MaxK || !fp4_format_ok(format) || !codes_ld || !scales_bytes)
    return ASHQK_ERR_INVALID_ARGUMENT;
  *codes_ld = fp4_padded_k(K) / 2;
  *scales_bytes = ceil_div64(M, kFp4TileRows) * fp4_scale_tiles(K, format) * kFp4TileBytes;
  return ASHQK_OK;
}

extern "C" int ashqk_quantize_fp4(const void* x, int64_t x_ld, int dtype, int gated, void* codes, int64_t codes_ld,
                                  void* scales, int M, int K, int format, float global_scale, void* stream) {
  const int size = dtype_size(dtype);
  if (!x || M <= 0 || K <= 0 || K > kFp4MaxK || !size || !aligned(x, size) || !fp4_format_ok(format))
    return ASHQK_ERR_INVALID_ARGUMENT;
  if (x_ld < static_cast<int64_t>(K) * (gated ? 2 : 1) || !fp4_global_scale_ok(format, global_scale))
    return ASHQK_ERR_INVALID_ARGUMENT;
  if (const int rc = check_fp4_operand(codes, codes_ld, scales, K)) return rc;
  return quantize_fp4({x, x_ld, dtype, gated != 0, global_scale}, static_cast<uint8_t*>(codes), codes_ld,
                      static_cast<uint8_t*>(scales), M, K, format, false, static_cast<cudaStream_t>(stream));
}

extern "C" int ashqk_dequantize_fp4(const void* codes, int64_t codes_ld, const void* scales, void* out, int64_t out_ld,
                                    int dtype, int M, int K, int format, float global_scale, void* stream) {
  const int size = dtype_size(dtype);
  if (!out || M <= 0 || K <= 0 || K > kFp4MaxK || !size || !aligned(out, size) || !fp4_format_ok(format))
    return ASHQK_ERR_INVALID_ARGUMENT;
  if (out_ld < K || !fp4_global_scale_ok(format, global_scale)) return ASHQK_ERR_INVALID_ARGUMENT;
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
