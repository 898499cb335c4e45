// The 4-bit format of weights and of cached keys and values: each group of
// consecutive elements of a row shares a bfloat16 scale
//   s = max(bf16(f32(max|x| / 7)), 2^-126),
// a code is the integer nearest to x / s (ties to even, the quotient taken
// exactly), -7 .. 7, stored as code + 8, and stands for code * s (exact in
// float32: 4 bits times 8).  The codes are formed with the rounded scale, so its
// rounding costs no accuracy.  A group with an infinity or a NaN gets s = NaN
// and codes 0 and decodes to NaN.  One finite value decodes to infinity, and in
// bfloat16 alone: its largest, 255 * 2^120, has s = 146 * 2^118 and stands for
// 1022 * 2^118, which lies halfway to 2^128 and rounds to that.
#pragma once
#include "esa_common.cuh"

namespace esa {
namespace int4 {

// Scale of a group whose largest magnitude has these float bits (NaN above infinity
// above finite), and its reciprocal to a unit in the last place.  a / 7 is rounded
// correctly by one step from q = a c, c the float32 nearest to 1 / 7, with the exact
// remainder a - 7 q (Markstein, IBM J. Res. Dev. 34, 1990).
__device__ __forceinline__ float group_scale(uint32_t top_bits, float& inv) {
  const float a = __uint_as_float(top_bits), c = 1.f / 7.f, q = a * c;
  float s = __bfloat162float(__float2bfloat16_rn(fmaf(fmaf(-7.f, q, a), c, q)));
  s = fmaxf(s, __uint_as_float(0x00800000u));
  if (top_bits >= 0x7f800000u) s = __uint_as_float(0x7fc00000u);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
  return s;
}

// 8 codes + 8 of a group of scale s, a nibble each.  The sum of an integer below 2^22
// and 1.5 * 2^23 has it as its low bits: the nibbles are put together by products of
// those words with powers of 16, what the constant part adds is taken out at the end.
// A group of scale NaN gets codes 0.
template <typename T>
__device__ __forceinline__ uint32_t codes_of(const float (&f)[8], float s, float inv) {
  constexpr float kMagic = 12582912.f + 8.f;
  uint32_t w = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float x = f[e], q = x * inv;
    float n;
    if constexpr (sizeof(T) == 2) {
      // x has 11 bits at most and s 8: the quotient is a half-integer exactly or at
      // least 2^-13 away from one, so its float32 rounding decides (ties to even)
      n = fmaf(fmaf(-q, s, x), inv, q) + kMagic;
    } else {
      // the remainder x - n s is exact (n s has 12 bits and lies next to x), so the
      // comparison with s / 2 settles what the quotient's rounding left open
      float i = rintf(q);
      const float r = fmaf(-i, s, x), a = 2.f * fabsf(r);
      if (a > s || (a == s && ((int)i & 1))) i += r > 0.f ? 1.f : -1.f;
      n = i + kMagic;
    }
    w += __float_as_uint(n) << (4 * e);
  }
  // sum of 0x4b400000 * 16^e over e < 8, modulo 2^32
  w -= 0x40000000u + 0xb4000000u + 0x4b400000u;
  return s == s ? w : 0x88888888u;
}

__device__ __forceinline__ float decode(uint32_t nibble, float s) {
  return (float)((int)(nibble & 15u) - 8) * s;
}

__device__ __forceinline__ uint32_t and_or(uint32_t w, uint32_t mask, uint32_t bits) {
  uint32_t v;          // (w & mask) | bits: written out, else it is two instructions
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(v) : "r"(w), "r"(mask), "r"(bits));
  return v;
}

// The values of the 8 nibbles of w (code + 8) in T, two (one) per word.  For bf16 the
// product of the code and the scale in bf16 is the rounding of their exact product;
// so for fp16 where the scale is one of its normal numbers.
template <typename T>
__device__ __forceinline__ void decode8(uint32_t w, float s, uint32_t (&out)[2 * sizeof(T)]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < 8; ++e) out[e] = __float_as_uint(decode(w >> (4 * e), s));
  } else {
    constexpr bool kHalf = std::is_same<T, __half>::value;
    uint32_t p[4];                          // nibbles j and j + 4
    if (kHalf && !(s >= 0x1p-14f && s <= 0x1p12f)) {
#pragma unroll
      for (int j = 0; j < 4; ++j) p[j] = Vec<T>::pack(decode(w >> (4 * j), s), decode(w >> (4 * j + 16), s));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        // 1024 + n (fp16) or 128 + n (bf16)
        const uint32_t v = and_or(w >> (4 * j), 0x000f000fu, kHalf ? 0x64006400u : 0x43004300u);
        if constexpr (kHalf) {
          const __half2 d = __hmul2(__hadd2(*reinterpret_cast<const __half2*>(&v), __float2half2_rn(-1032.f)),
                                    __float2half2_rn(s));
          p[j] = *reinterpret_cast<const uint32_t*>(&d);
        } else {
          const __nv_bfloat162 d =
              __hmul2(__hadd2(*reinterpret_cast<const __nv_bfloat162*>(&v), __float2bfloat162_rn(-136.f)),
                      __float2bfloat162_rn(s));
          p[j] = *reinterpret_cast<const uint32_t*>(&d);
        }
      }
    }
    out[0] = __byte_perm(p[0], p[1], 0x5410);
    out[1] = __byte_perm(p[2], p[3], 0x5410);
    out[2] = __byte_perm(p[0], p[1], 0x7632);
    out[3] = __byte_perm(p[2], p[3], 0x7632);
  }
}

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

}  // namespace int4
}  // namespace esa
