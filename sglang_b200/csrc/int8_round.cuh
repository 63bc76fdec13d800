// Rounding to symmetric 8-bit integers, the same wherever rows are quantised.
#pragma once

#include "common.cuh"

namespace b200 {

// max that keeps a NaN: a row must not hide one behind its other values
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// The nearest whole number of |v| < 2^22, ties to even, in the low bits of the result: adding 1.5 * 2^23 leaves no room for a fraction.
__device__ __forceinline__ uint32_t rint_bits(float v) { return __float_as_uint(v + 12582912.f); }

// x / s rounded to the nearest float, r = 1 / s rounded: one residual step (Markstein)
__device__ __forceinline__ float div_by(float x, float s, float r) {
  const float q = x * r;
  return fmaf(fmaf(-q, s, x), r, q);
}

// Eight codes, rint_bits() of each value, as bytes
__device__ __forceinline__ uint2 pack8_s8(const uint32_t (&c)[8]) {
  uint2 out;
  out.x = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
  out.y = __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410);
  return out;
}

// Scale of 8-bit integers for a largest magnitude
__device__ __forceinline__ float int8_scale(float amax) { return __fdiv_rn(max_nan(amax, 1e-10f), 127.f); }

}  // namespace b200
