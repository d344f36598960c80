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

constexpr int kFp4TileRows = 128;
constexpr int kFp4TileBytes = 512;

inline bool fp4_format_ok(int format) { return format == ASHQK_MXFP4 || format == ASHQK_NVFP4; }
__host__ __device__ constexpr int fp4_block(int format) { return format == ASHQK_MXFP4 ? 32 : 16; }
__host__ __device__ constexpr int64_t fp4_padded_k(int64_t k) { return (k + 31) / 32 * 32; }
// Tiles of four scales along a row.
__host__ __device__ constexpr int64_t fp4_scale_tiles(int64_t k, int format) {
  return (fp4_padded_k(k) / fp4_block(format) + 3) / 4;
}
__device__ __forceinline__ int64_t fp4_scale_offset(int64_t row, int block, int64_t tiles) {
  return ((row >> 7) * tiles + (block >> 2)) * kFp4TileBytes + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (block & 3);
}

// What a quantiser needs of the global scale g; on the host.
struct Fp4Quant {
  float gs, six_gs, inv_six_gs;  // g, 6 g and 1 / (6 g), each rounded to fp32
};
inline Fp4Quant fp4_quant_params(float gs) {
  const float six = 6.0f * gs;
  return {gs, six, 1.0f / six};
}

// v / d, rounded to fp32 as one division is, from r = 1 / d correctly rounded: the product v r is off by at most a
// unit in the last place, and one step with the exact residual corrects it (P. W. Markstein, Computation of
// elementary functions on the IBM RISC System/6000 processor, IBM J. Res. Dev. 34, 1990). Quotients are cut
// off at +-1024, beyond what either format holds, so that the residual stays finite.
__device__ __forceinline__ float quotient(float v, float d, float r) {
  const float q = fminf(fmaxf(v * r, -1024.0f), 1024.0f);
  return fmaf(fmaf(-q, d, v), r, q);
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
    *r = *d > 0.0f ? __frcp_rn(*d) : 0.0f;
    return byte;
  }
}

// A value over its scale, before rounding to E2M1. For NVFP4 the rounded quotient and not the product with the
// reciprocal, which would move exact ties (x = 0.75 d, which 16-bit inputs meet often) off the border.
template <int FMT>
__device__ __forceinline__ float fp4_scaled(float v, float d, float r) {
  return FMT == ASHQK_MXFP4 ? v * r : quotient(v, d, r);
}

// Eight scaled values -> eight E2M1 codes, the first in the lowest four bits; to nearest even, held
// to +-6.
__device__ __forceinline__ uint32_t fp4_pack8(const float (&v)[8]) {
  uint32_t r;
  asm("{\n"
      " .reg .b8 b0, b1, b2, b3;\n"
      " cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n"
      " cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n"
      " cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n"
      " cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n"
      " mov.b32 %0, {b0, b1, b2, b3};\n"
      "}\n"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}

// Eight E2M1 codes -> values.
__device__ __forceinline__ void fp4_unpack8(uint32_t codes, float (&v)[8]) {
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

// Eight consecutive 16-bit values as they lie in memory: `vec` when p is 16-byte aligned and all eight exist, else
// one by one with zeros from `count` on.
template <typename T>
__device__ __forceinline__ uint4 load8_raw(const T* p, int count, bool vec) {
  static_assert(sizeof(T) == 2, "16-bit types");
  if (vec) return ld_once_v4(p);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint16_t* h = reinterpret_cast<const uint16_t*>(p) + 2 * i;
    w[i] = (2 * i < count ? h[0] : 0u) | ((2 * i + 1 < count ? h[1] : 0u) << 16);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <typename T>
__device__ __forceinline__ void unpack8(const uint4& u, float (&v)[8]) {
  unpack2<T>(u.x, v[0], v[1]);
  unpack2<T>(u.y, v[2], v[3]);
  unpack2<T>(u.z, v[4], v[5]);
  unpack2<T>(u.w, v[6], v[7]);
}
template <typename T>
__device__ __forceinline__ void load8(const T* p, int count, bool vec, float (&v)[8]) {
  if constexpr (sizeof(T) == 2) {
    unpack8<T>(load8_raw(p, count, vec), v);
  } else if (vec) {
    const uint4 a = ld_once_v4(p), b = ld_once_v4(p + 4);
    v[0] = __uint_as_float(a.x), v[1] = __uint_as_float(a.y), v[2] = __uint_as_float(a.z), v[3] = __uint_as_float(a.w);
    v[4] = __uint_as_float(b.x), v[5] = __uint_as_float(b.y), v[6] = __uint_as_float(b.z), v[7] = __uint_as_float(b.w);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < count ? p[i] : 0.0f;
  }
}

// silu(gate) * up in fp32. exp overflows to infinity for gates below -88 and the quotient is then 0.
__device__ __forceinline__ float silu_mul(float gate, float up) {
  return __fdividef(gate, 1.0f + __expf(-gate)) * up;
}

// The largest magnitude of eight 16-bit values, as the fp32 bit pattern of its absolute value.
template <typename T>
__device__ __forceinline__ uint32_t abs_max8_raw(const uint4& u) {
  uint32_t m = __vmaxu2(__vmaxu2(u.x & 0x7fff7fffu, u.y & 0x7fff7fffu), __vmaxu2(u.z & 0x7fff7fffu, u.w & 0x7fff7fffu));
  m = max(m & 0xffffu, m >> 16);
  if constexpr (std::is_same_v<T, __nv_bfloat16>)
    return m << 16;
  else
    return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(m))));
}

// The largest bit pattern of |v|: as an unsigned number it orders finite < infinity < NaN.
__device__ __forceinline__ uint32_t abs_max8(const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
  return m;
}

}  // namespace ashqk
