// Rounding to symmetric 8-bit integers, the same wherever rows are quantised.
#pragma once

#include "common.cuh"

namespace b200 {

// griddepcontrol.wait, and a zero that is known only behind it: added to an operand's address it keeps the loads there, which the compiler
// may otherwise move as it likes. They are ordinary loads, which the wait covers, and not from the read-only path: an earlier kernel of
// the stream may have written the operand while this one was already resident.
__device__ __forceinline__ int64_t grid_dependency_zero() {
  int64_t zero;
  asm volatile("griddepcontrol.wait;\n\tmov.b64 %0, 0;" : "=l"(zero)::"memory");
  return zero;
}
__device__ __forceinline__ uint4 ld_again_16(const void* p) {  // read by every row
  uint4 v;
  asm("ld.global.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

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

__device__ __forceinline__ uint64_t twice(float v) {
  uint64_t p;
  asm("mov.b64 %0, {%1, %1};" : "=l"(p) : "f"(v));
  return p;
}

// rint_bits of a product that is not rounded before, and of two at once
__device__ __forceinline__ uint32_t rint_scaled(float y, float scale) { return __float_as_uint(fmaf(y, scale, 12582912.f)); }
__device__ __forceinline__ void rint_scaled_two(float y0, float y1, uint64_t scale, uint32_t& c0, uint32_t& c1) {
  asm("{.reg .b64 y; mov.b64 y, {%2, %3}; fma.rn.f32x2 y, y, %4, %5; mov.b64 {%0, %1}, y;}"
      : "=r"(c0), "=r"(c1)
      : "f"(y0), "f"(y1), "l"(scale), "l"(twice(12582912.f)));
}

// Two quotients at once, as div_by gives them, and their nearest whole numbers: half the instructions, which had bounded the quantiser of
// long prefills (8192 x 14336 bf16: 73 % of the issue slots at 5.8 TB/s; 16384 x 8192 70.5 -> 63.5 us).
struct DivTwo {
  uint64_t minus_s, r, magic;
  __device__ __forceinline__ DivTwo(float s, float inv) : minus_s(twice(-s)), r(twice(inv)), magic(twice(12582912.f)) {}
  __device__ __forceinline__ void rint_bits(float x0, float x1, uint32_t& c0, uint32_t& c1) const {
    asm("{\n\t"
        ".reg .b64 x, q, e;\n\t"
        "mov.b64 x, {%2, %3};\n\t"
        "mul.rn.f32x2 q, x, %5;\n\t"
        "fma.rn.f32x2 e, q, %4, x;\n\t"
        "fma.rn.f32x2 q, e, %5, q;\n\t"
        "add.rn.f32x2 q, q, %6;\n\t"
        "mov.b64 {%0, %1}, q;\n\t"
        "}"
        : "=r"(c0), "=r"(c1)
        : "f"(x0), "f"(x1), "l"(minus_s), "l"(r), "l"(magic));
  }
};

// Eight codes, rint_bits() of each value, as bytes
__device__ __forceinline__ uint2 pack8_s8(const uint32_t (&c)[8]) {
  uint2 out;
  out.x = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
  out.y = __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410);
  return out;
}

// m / 127 as IEEE rounds it: one residual step does so for every mantissa; infinities and NaN stay
__device__ __forceinline__ float over_127(float m) { return m < INFINITY ? div_by(m, 127.f, 1.f / 127.f) : m; }

// Scale of 8-bit integers for a largest magnitude
__device__ __forceinline__ float int8_scale(float amax) { return over_127(max_nan(amax, 1e-10f)); }

}  // namespace b200
