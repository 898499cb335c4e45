// The 4-bit format of weights and of cached keys and values: each group of
// consecutive elements of a row shares a bfloat16 scale
//   s = max(bf16(f32(max|x| / 7)), 2^-126),
// a code is the integer nearest to x / s (ties to even, the quotient taken
// exactly), -7 .. 7, stored as code + 8, and stands for code * s (exact in
// float32: 4 bits times 8).  The codes are formed with the rounded scale, so its
// rounding costs no accuracy.  A group with an infinity or a NaN gets s = NaN
// and codes 0 and decodes to NaN.
#pragma once
#include "esa_common.cuh"

namespace esa {
namespace int4 {

// Scale of a group whose largest magnitude has these float bits (NaN above
// infinity above finite).
__device__ __forceinline__ float group_scale(uint32_t top_bits) {
  if (top_bits >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  const float s = __bfloat162float(__float2bfloat16_rn(__fdiv_rn(__uint_as_float(top_bits), 7.f)));
  return fmaxf(s, __uint_as_float(0x00800000u));
}

// code + 8 of x in a group of scale s with inv about 1 / s.
__device__ __forceinline__ uint32_t code_of(float x, float s, float inv) {
  if (s != s) return 8u;
  float n = rintf(x * inv);
  // the remainder x - n s is exact (n s has 12 bits, and lies next to x), so the
  // comparison with s / 2 settles what the product's rounding left open
  const float r = fmaf(-n, s, x), a = 2.f * fabsf(r);
  const bool odd = ((int)n & 1) != 0;
  if (a > s || (a == s && odd)) n += r > 0.f ? 1.f : -1.f;
  return (uint32_t)((int)n + 8);
}

__device__ __forceinline__ float decode(uint32_t nibble, float s) {
  return (float)((int)(nibble & 15u) - 8) * s;
}

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

}  // namespace int4
}  // namespace esa
