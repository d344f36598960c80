// Microscaled 4-bit floating point: the two formats, their memory layout and the
// rounding of values into them.
//
// An element is E2M1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and negatives); blocks of a row's columns share a
// scale. ASHQK_MXFP4: 32 columns, scale 2^(floor(log2 amax) - 2) as E8M0. ASHQK_NVFP4: 16 columns,
// scale E4M3(min(448, amax / (6 g))) times the tensor's global scale g.
//
// Codes: two to a byte, the even column low; a row holds Kp = K rounded up to 32 columns, the padding
// zero, so that a row pitch is a multiple of 16 bytes (what TMA asks of a row stride). Scales: tiles of
// 128 rows x 4 blocks, 512 bytes each, [row tile][block tile][row % 32][row / 32 % 4][block % 4] --
// the byte order in which tcgen05.cp (32x128b, broadcast to the four lane quarters) lays a tile
// down in four TMEM columns as the block-scaled MMA reads it, so a kernel copies tiles and shuffles
// nothing. Padding blocks of a tile hold scale byte 0; padding rows hold anything.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"

namespace ashqk {

constexpr int kFp4MaxK = 1 << 24;        // columns; offsets within 128 rows of codes stay below 2^31
constexpr int64_t kFp4MaxLd = 1 << 24;   // bytes from row to row of codes
constexpr int kFp4TileRows = 128;
constexpr int kFp4TileBytes = 512;

inline bool fp4_format_ok(int format) { return format == ASHQK_MXFP4 || format == ASHQK_NVFP4; }
__host__ __device__ constexpr int fp4_block(int format) { return format == ASHQK_MXFP4 ? 32 : 16; }
__host__ __device__ constexpr int64_t fp4_padded_k(int64_t k) { return (k + 31) / 32 * 32; }
// Tiles of four scales along a row.
__host__ __device__ constexpr int64_t fp4_scale_tiles(int64_t k, int format) {
  return (fp4_padded_k(k) / fp4_block(format) + 3) / 4;
}
// Offset of the scale of (row, block); I: 32 or 64 bits.
template <typename I>
__device__ __forceinline__ I fp4_scale_offset(I row, uint32_t block, I tiles) {
  return ((row >> 7) * tiles + (block >> 2)) * kFp4TileBytes + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (block & 3);
}

// ---- the host functions that the files share ----------------------------------------------------

// A quantised matrix of `rows` rows.
struct Fp4Matrix {
  const uint8_t* codes;
  int64_t ld;
  const uint8_t* scales;
  int rows;
};
// y [a.rows, b.rows] = alpha * a b^T; dtype F16 or BF16.
struct Fp4Product {
  Fp4Matrix a, b;
  int K, format;
  float alpha;
  void* y;
  int64_t y_ld;
  int dtype;
};
// What is to be quantised: 16- or 32-bit rows, gated or not.
struct Fp4Source {
  const void* x;
  int64_t ld;
  int dtype;
  bool gated;
  float gs;
};

int dtype_size(int dtype);  // 0: no such type
int check_fp4_operand(const void* codes, int64_t codes_ld, const void* scales, int K);
bool fp4_global_scale_ok(int format, float gs);
// `early`: let the next launch start while this one runs. Only for a consumer that reads the result
// behind its own griddepcontrol.wait.
int quantize_fp4(const Fp4Source& x, uint8_t* codes, int64_t codes_ld, uint8_t* scales, int M, int K, int format, bool early,
                 cudaStream_t stream);
int fp4_matmul_rows(const Fp4Product& p, cudaStream_t stream);
int fp4_matmul_pair(const Fp4Product& p, cudaStream_t stream);
bool fp4_fused_ok(int M, int N, int K, bool gated);
// p.a is not used but for its rows.
int fp4_linear_rows(const Fp4Source& x, const Fp4Product& p, cudaStream_t stream);
void fp4_set_pair_split(int split);

// What a quantiser needs of the global scale g; on the host.
struct Fp4Quant {
  float gs, six_gs, inv_six_gs;  // g, 6 g and 1 / (6 g), each rounded to fp32
};
inline Fp4Quant fp4_quant_params(float gs) {
  const float six = 6.0f * gs;
  return {gs, six, 1.0f / six};
}

// v / d from an r near 1 / d (within two units in the last place): the product v r, corrected once by the exact
// residual, differs from the quotient rounded once only where that lies within 2^-20 units of halfway between two
// fp32 values -- never where the quotient is an fp32 value, as the borders between codes are (after
// P. W. Markstein, Computation of elementary functions on the IBM RISC System/6000 processor, IBM J. Res.
// Dev. 34, 1990). Quotients are cut off at +-1024, beyond what either format holds, so that the residual
// stays finite.
__device__ __forceinline__ float quotient(float v, float d, float r) {
  const float q = fminf(fmaxf(v * r, -1024.0f), 1024.0f);
  return fmaf(fmaf(-q, d, v), r, q);
}
__device__ __forceinline__ float reciprocal_approx(float d) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
  return r;
}

// The scale of a block whose largest magnitude has the fp32 bit pattern `amax` (sign cleared): its byte, its value d
// and 1 / d. A block that holds an infinity or a NaN (the pattern compares above every finite one) gets the
// format's NaN scale. A scale of zero (NVFP4, a tiny block) comes with a reciprocal of zero.
template <int FMT>
__device__ __forceinline__ uint32_t fp4_scale_of(uint32_t amax, const Fp4Quant& q, float* d, float* r) {
  if (FMT == ASHQK_MXFP4) {
    // Exponent field E of amax; the scale's is E - 2, not below 0 (2^-127). Its inverse 2^(127 - byte) is exact.
    const uint32_t e = amax >> 23;
    const uint32_t byte = amax >= 0x7f800000u ? 255u : (e > 2u ? e - 2u : 0u);
    *d = 0.0f;  // not used
    *r = __uint_as_float((254u - (byte == 255u ? 254u : byte)) << 23);
    return byte;
  } else {
    const float t = quotient(__uint_as_float(amax), q.six_gs, q.inv_six_gs);
    uint16_t pair;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(pair) : "f"(0.0f), "f"(t));
    const uint32_t byte = amax >= 0x7f800000u ? 0x7fu : (pair & 0x7fu);
    uint32_t h2;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"(static_cast<uint16_t>(byte)));
    *d = __low2float(u32_as_h2(h2)) * q.gs;
    *r = *d > 0.0f ? reciprocal_approx(*d) : 0.0f;
    return byte;
  }
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ uint64_t f32x2(float lo, float hi) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
  return v;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}

// Four pairs of scaled values -> eight E2M1 codes, the first in the lowest four bits; to nearest even, held to +-6.
__device__ __forceinline__ uint32_t fp4_pack8(const uint64_t* v) {
  uint32_t r;
  asm("{\n"
      " .reg .b8 b0, b1, b2, b3;\n"
      " .reg .f32 l, h;\n"
      " mov.b64 {l, h}, %1;\n"
      " cvt.rn.satfinite.e2m1x2.f32 b0, h, l;\n"
      " mov.b64 {l, h}, %2;\n"
      " cvt.rn.satfinite.e2m1x2.f32 b1, h, l;\n"
      " mov.b64 {l, h}, %3;\n"
      " cvt.rn.satfinite.e2m1x2.f32 b2, h, l;\n"
      " mov.b64 {l, h}, %4;\n"
      " cvt.rn.satfinite.e2m1x2.f32 b3, h, l;\n"
      " mov.b32 %0, {b0, b1, b2, b3};\n"
      "}\n"
      : "=r"(r)
      : "l"(v[0]), "l"(v[1]), "l"(v[2]), "l"(v[3]));
  return r;
}

// The codes of sixteen values that share the scale fp4_scale_of gave.
//
// For NVFP4 a code is the corrected quotient's, by quotient()'s arithmetic in pairs, and not that of the product with
// the reciprocal, which would move exact ties (x = 0.75 d, which 16-bit inputs meet often) off the border.
template <int FMT>
__device__ __forceinline__ uint2 fp4_codes16(float* v, uint32_t byte, float d, float r) {
  if (FMT == ASHQK_NVFP4 && byte == 126u) {  // perhaps beyond the largest scale: quotients without bound
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = fminf(fmaxf(v[i], -8.0f * d), 8.0f * d);
  }
  const uint64_t r2 = f32x2(r, r), nd2 = f32x2(-d, -d);
  uint64_t s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint64_t x = f32x2(v[2 * i], v[2 * i + 1]);
    s[i] = mul2(x, r2);
    if (FMT == ASHQK_NVFP4) s[i] = fma2(fma2(s[i], nd2, x), r2, s[i]);
  }
  return make_uint2(fp4_pack8(s), fp4_pack8(s + 4));
}

// Sixteen values of one block (NVFP4) or of half a block whose other half the neighbouring lane has (MXFP4) -> their
// codes and the block's scale byte. `amax`: the largest magnitude of these sixteen, as fp32 bits. All lanes of
// the warp call it together.
template <int FMT>
__device__ __forceinline__ uint32_t fp4_quantize16(float (&v)[16], uint32_t amax, const Fp4Quant& q, uint2* codes) {
  if (FMT == ASHQK_MXFP4) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
  float d, r;
  const uint32_t byte = fp4_scale_of<FMT>(amax, q, &d, &r);
  *codes = fp4_codes16<FMT>(v, byte, d, r);
  return byte;
}

// Eight E2M1 codes -> values.
__device__ __forceinline__ void fp4_unpack8(uint32_t codes, float* v) {
  uint32_t h[4];
  asm("{\n"
      " .reg .b8 b0, b1, b2, b3;\n"
      " mov.b32 {b0, b1, b2, b3}, %4;\n"
      " cvt.rn.f16x2.e2m1x2 %0, b0;\n"
      " cvt.rn.f16x2.e2m1x2 %1, b1;\n"
      " cvt.rn.f16x2.e2m1x2 %2, b2;\n"
      " cvt.rn.f16x2.e2m1x2 %3, b3;\n"
      "}\n"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(codes));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(u32_as_h2(h[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

// The fp32 value of a scale byte, without the global scale.
template <int FMT>
__device__ __forceinline__ float fp4_scale_value(uint32_t byte) {
  if (FMT == ASHQK_MXFP4) {
    if (byte == 255u) return __uint_as_float(0x7fffffffu);
    return byte ? __uint_as_float(byte << 23) : __uint_as_float(0x00400000u);  // 2^-127 is subnormal
  } else {
    uint32_t h2;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"(static_cast<uint16_t>(byte)));
    return __low2float(u32_as_h2(h2));
  }
}

// ---- element types of inputs and outputs ------------------------------------------------------

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) { return h2_as_u32(__floats2half2_rn(lo, hi)); }
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

template <typename T>
__device__ __forceinline__ void unpack2(uint32_t u, float& lo, float& hi);
template <>
__device__ __forceinline__ void unpack2<__half>(uint32_t u, float& lo, float& hi) {
  const float2 f = __half22float2(u32_as_h2(u));
  lo = f.x;
  hi = f.y;
}
template <>
__device__ __forceinline__ void unpack2<__nv_bfloat16>(uint32_t u, float& lo, float& hi) {
  lo = __uint_as_float(u << 16);
  hi = __uint_as_float(u & 0xffff0000u);
}

// Read once, and not through the read-only path: with programmatic dependent launch the previous kernel may still be
// writing when this one starts.
__device__ __forceinline__ uint4 ld_once_v4(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p)
               : "memory");
  return v;
}

// Sixteen consecutive values as they lie in memory. `align`: what the caller knows of the address, 32 or 16 bytes, and
// then all sixteen exist; else 0, and of the values those from `count` on read as zero. Without alignment the
// 16-byte granules that hold the values are loaded whole (a granule with a byte of an allocation is in it) and
// shifted into place.
template <typename T>
struct Raw16 {
  uint32_t w[4 * sizeof(T)];
};
template <typename T>
__device__ __forceinline__ void load16(const T* p, int count, int align, Raw16<T>& r) {
  constexpr int kWords = 4 * sizeof(T);
  if (align == 32) {
#pragma unroll
    for (int i = 0; i < kWords; i += 8)
      asm volatile("ld.global.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                   : "=r"(r.w[i]), "=r"(r.w[i + 1]), "=r"(r.w[i + 2]), "=r"(r.w[i + 3]), "=r"(r.w[i + 4]),
                     "=r"(r.w[i + 5]), "=r"(r.w[i + 6]), "=r"(r.w[i + 7])
                   : "l"(reinterpret_cast<const uint32_t*>(p) + i)
                   : "memory");
  } else if (align == 16) {
#pragma unroll
    for (int i = 0; i < kWords; i += 4) {
      const uint4 u = ld_once_v4(reinterpret_cast<const uint32_t*>(p) + i);
      r.w[i] = u.x, r.w[i + 1] = u.y, r.w[i + 2] = u.z, r.w[i + 3] = u.w;
    }
  } else {
    const uintptr_t first = reinterpret_cast<uintptr_t>(p), last = first + sizeof(T) * min(count, 16);
    const uint32_t off = first & 15u;
    uint32_t w[kWords + 4];
#pragma unroll
    for (int i = 0; i < kWords + 4; i += 4) {
      const uintptr_t at = first - off + 4 * i;
      const uint4 u = at < last ? ld_once_v4(reinterpret_cast<const void*>(at)) : make_uint4(0, 0, 0, 0);
      w[i] = u.x, w[i + 1] = u.y, w[i + 2] = u.z, w[i + 3] = u.w;
    }
#pragma unroll
    for (int i = 0; i < kWords + 3; ++i) w[i] = off & 4u ? w[i + 1] : w[i];
#pragma unroll
    for (int i = 0; i < kWords + 1; ++i) w[i] = off & 8u ? w[i + 2] : w[i];
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      if constexpr (sizeof(T) == 2) {
        r.w[i] = off & 2u ? __funnelshift_r(w[i], w[i + 1], 16) : w[i];
        if (2 * i + 1 >= count) r.w[i] = 2 * i < count ? r.w[i] & 0xffffu : 0u;
      } else {
        r.w[i] = i < count ? w[i] : 0u;
      }
    }
  }
}
// What is known of the address of column 16 j for every row of a matrix.
inline int chunk_align(const void* p, int64_t ld, int size) {
  return aligned(p, 32) && ld * size % 32 == 0 ? 32 : aligned(p, 16) && ld * size % 16 == 0 ? 16 : 0;
}

template <typename T>
__device__ __forceinline__ void unpack16(const Raw16<T>& r, float* v) {
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < 8; ++i) unpack2<T>(r.w[i], v[2 * i], v[2 * i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r.w[i]);
  }
}

// The largest magnitude, as fp32 bits: as an unsigned number those order finite < infinity < NaN.
__device__ __forceinline__ uint32_t abs_max16(const float* v) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
  return m;
}
template <typename T>
__device__ __forceinline__ uint32_t abs_max16(const Raw16<T>& r) {
  if constexpr (sizeof(T) == 2) {  // 16-bit patterns have the same order
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = __vmaxu2(m, r.w[i] & 0x7fff7fffu);
    m = max(m & 0xffffu, m >> 16);
    if constexpr (std::is_same_v<T, __nv_bfloat16>)
      return m << 16;
    else
      return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(m))));
  } else {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) m = max(m, r.w[i] & 0x7fffffffu);
    return m;
  }
}

// 2^x; results below 2^-126 are 0.
__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
constexpr float kLog2E = 1.44269504088896341f;

// silu(gate) * up in fp32: gate / (1 + exp(-gate)) times up for gates from -80 on, where the denominator and its reciprocal
// are normal numbers. Below, where 1 + exp(gate) is 1 in fp32 but exp(-gate) soon overflows, with h = exp(gate / 2) as
// (gate h) (up h): each factor h meets an operand first, so nothing vanishes on the way while the result is a normal
// number. Relative error at most 2^-20 + 2^-23 |gate|: the exponent's rounding and its constant's (1.25 |gate| 2^-24), two
// units of the exponential (twice where h is), one of the reciprocal, at most four roundings. Gates below -174 give 0 (less
// than 2^-116 in truth).
__device__ __forceinline__ float silu_mul_any(float gate, float up) {
  if (gate < -80.0f) {
    const float h = exp2_approx(gate * (0.5f * kLog2E));
    return (gate * h) * (up * h);
  }
  return gate * reciprocal_approx(1.0f + exp2_approx(gate * -kLog2E)) * up;
}
// Sixteen values, v[i] = silu(v[i]) * up[i]. Gates below -80 are rare: a thread that has none multiplies in pairs (8192 x
// 12288 to MXFP4, L2 warm: 71.3 us, one by one 72.4).
__device__ __forceinline__ void silu_mul16(float* v, const float* up) {
  float least = v[0];
#pragma unroll
  for (int i = 1; i < 16; ++i) least = fminf(least, v[i]);
  if (least >= -80.0f) {
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      const uint64_t g = f32x2(v[i], v[i + 1]);
      float t0, t1;
      asm("mov.b64 {%0, %1}, %2;" : "=f"(t0), "=f"(t1) : "l"(mul2(g, f32x2(-kLog2E, -kLog2E))));
      const uint64_t r =
          f32x2(reciprocal_approx(1.0f + exp2_approx(t0)), reciprocal_approx(1.0f + exp2_approx(t1)));
      asm("mov.b64 {%0, %1}, %2;" : "=f"(v[i]), "=f"(v[i + 1]) : "l"(mul2(mul2(g, r), f32x2(up[i], up[i + 1]))));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = silu_mul_any(v[i], up[i]);
  }
}

}  // namespace ashqk
