// e4m3 rows with one scale for each block of 128: the rule that every kernel writing such rows uses.
// A block's scale is the smallest power of two that brings its values within 448, the largest e4m3
// value: dividing by it is exact, so a value is rounded once, to e4m3.  A block of zeros has the scale 1; a
// block with an infinity or a NaN has the scale NaN, so that whatever is computed from it is NaN.
#pragma once

#include "common.cuh"

namespace xdit {

constexpr int kBlock = XDIT_FP8_BLOCK;

// The larger of two absolute values; a NaN wins.
__device__ __forceinline__ float amax_nan(float m, float x) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(m), "f"(fabsf(x)));
  return r;
}
// The largest of m and two absolute values (m is one already); a NaN wins.
__device__ __forceinline__ float amax_nan(float m, float x, float y) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(m), "f"(x), "f"(y));
  return r;
}
// Scale of a block whose largest magnitude is `top`, and its reciprocal (both powers of two).
__device__ __forceinline__ float block_scale(float top, float& inverse) {
  const uint32_t bits = __float_as_uint(top);
  int e = (int)(bits >> 23) - 8;                 // biased exponent of the scale: 448 = 1.75 * 2^8
  if ((bits & 0x7fffffu) > 0x600000u) ++e;       // mantissa above 1.75
  if (e < 1) e = 1;                              // smallest normal power of two: its reciprocal is finite
  float s = __uint_as_float((uint32_t)e << 23);
  float i = __uint_as_float((uint32_t)(254 - e) << 23);
  if (top == 0.f) { s = 1.f; i = 1.f; }
  if (!(top <= 3.402823466e38f)) s = i = __uint_as_float(0x7fc00000u);
  inverse = i;
  return s;
}
// Four values -> four e4m3 bytes, round to nearest even (the inputs are within 448, or NaN).
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return (uint32_t)lo | ((uint32_t)hi << 16);
}

}  // namespace xdit
