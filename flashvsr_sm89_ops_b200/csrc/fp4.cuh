// Microscaled 4-bit floating point: E2M1 codes with a scale per block of a row.
//
//   mx  blocks of 32, scale 2^e (E8M0 byte e + 127), e = floor(log2 amax) - 2
//   nv  blocks of 16, scale E4M3(amax / (6 r)), r one fp32 power of two per row: the smallest
//       2^k with row amax <= 448 * 6 * 2^k (k >= -100), so block scales use E4M3's whole range
//   code = E2M1(x / scale), to nearest, ties to even, saturating at 6
//
// r is a power of two so that every decision is exact in fp32: x / r is exact, and a block
// scale or a code is decided by comparing a quotient with a midpoint of a few bits.  An fp32
// x = m s (1 + d) with d != 0 differs from the midpoint product m s by at least one ulp of x,
// and the rounded quotient then differs from m (s has at most 4 significant bits), so the
// rounded quotient sits on a midpoint only when the exact one does.
// A non-finite value counts as 0 in the maxima and makes its block's scale NaN (0xFF / 0x7F),
// so the whole block stands for NaN.
//
// Layout: codes two to a byte, even element in the low nibble, rows padded with zero codes to
// a multiple of 32 elements (16 bytes, what TMA asks of a row pitch).  Block scale j of row m
// is byte (m % 32) * 16 + (m % 128) / 32 * 4 + j % 4 of the 512-byte tile (m / 128, j / 4),
// tiles row-major: the order in which the tensor core wants 128 rows' scales in TMEM, so a
// tile goes global -> shared -> TMEM as it is.  Scales past a row's last block are 0.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

namespace fvb {
namespace fp4 {

__host__ __device__ constexpr int block_elems(int fmt) { return fmt == FVB_FP4_NV ? 16 : 32; }
// bytes of one row of codes / 512-byte scale tiles along one row
inline int64_t code_pitch(int64_t K) { return (K + 31) / 32 * 16; }
__host__ __device__ inline int64_t scale_tiles(int64_t K, int fmt) {
  const int per = 4 * block_elems(fmt);
  return (K + per - 1) / per;
}

// byte of block scale (m, j) in its buffer of `tiles` tiles per row of tiles
__device__ __forceinline__ int64_t scale_at(int64_t m, int64_t j, int64_t tiles) {
  return ((m >> 7) * tiles + (j >> 2)) * 512 + (m & 31) * 16 + ((m & 127) >> 5) * 4 + (j & 3);
}

// max(m, |x.lo|, |x.hi|), a NaN if one is
__device__ __forceinline__ float max_abs_nan(float m, uint64_t x) {
  float a, b, r;
  f2_unpack(x, a, b);
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(m), "f"(fabsf(a)), "f"(fabsf(b)));
  return r;
}

// 8 fp32 -> 8 E2M1 codes (nearest even, saturating), element 0 in the low nibble
__device__ __forceinline__ uint32_t e2m1x8(const float* v) {
  uint32_t r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}

// 8 E2M1 codes -> 4 x f16x2 (exact)
__device__ __forceinline__ void e2m1x8_to_f16(uint32_t c, uint32_t* h) {
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "mov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(c));
}

// 2^e for e in [-127, 127] (2^-127 is subnormal)
__device__ __forceinline__ float pow2i(int e) {
  return __uint_as_float(e > -127 ? (uint32_t)(e + 127) << 23 : 1u << 22);
}

// the row scale's exponent from the row's finite amax: the smallest k >= -100 with
// amax <= 2688 * 2^k (2688 = 1.3125 * 2^11: carry into the exponent when the mantissa is above)
__device__ __forceinline__ int row_exponent(float amax) {
  const uint32_t b = __float_as_uint(amax);
  const int k = (int)((b + (0x7FFFFFu - 0x280000u)) >> 23) - 138;
  return b == 0u ? 0 : (k < -100 ? -100 : k);
}

// floor(log2 amax) - 2 in [-127, 127]; -127 for 0
__device__ __forceinline__ int mx_exponent(float amax) {
  const uint32_t b = __float_as_uint(amax);
  // subnormals (|x| < 2^-126) end at the clamp whatever their exponent
  const int e = (int)(b >> 23) - 129;
  return e < -127 ? -127 : e;
}

// x / d to the exact side of every midpoint: one correction of x * r, r = 1 / d rounded
__device__ __forceinline__ float quotient(float x, float d, float r) {
  const float q = x * r;
  return __fmaf_rn(__fmaf_rn(-q, d, x), r, q);
}

// E4M3 code of amax / (6 * 2^k); ik = 2^-k
__device__ __forceinline__ uint32_t nv_scale(float amax, float ik) {
  return f32_to_e4m3(quotient(amax * ik, 6.0f, 1.0f / 6.0f));
}
__device__ __forceinline__ float e4m3_value(uint32_t c) {
  const __half_raw h = __nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)c, __NV_E4M3);
  return __half2float(__half(h));
}

// codes of 16 values with one nv scale (E4M3 code c, row scale 2^k = rs)
__device__ __forceinline__ uint2 nv_codes16(const float* f, uint32_t c, float rs) {
  const float d = e4m3_value(c) * rs;
  float q[16];
  if (c == 0u) {
#pragma unroll
    for (int i = 0; i < 16; ++i) q[i] = 0.0f * f[i];
  } else {
    const float r = __frcp_rn(d);
#pragma unroll
    for (int i = 0; i < 16; ++i) q[i] = quotient(f[i], d, r);
  }
  return make_uint2(e2m1x8(q), e2m1x8(q + 8));
}
// codes of 16 values with an mx scale 2^e: the division is a power-of-two product, exact
__device__ __forceinline__ uint2 mx_codes16(const float* f, int e) {
  const float r = pow2i(-e);
  float q[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) q[i] = f[i] * r;
  return make_uint2(e2m1x8(q), e2m1x8(q + 8));
}

}  // namespace fp4
}  // namespace fvb
