// Activations kept in 8 bits between the forward and the backward pass.
//
// Each group of 128 consecutive elements of a row (the last group of a row
// may be shorter) shares one float32 scale s; with a = max |x| of the group:
//
//   int8:  s = max(f32(a / 127), 2^-126),  code = x / s rounded to the nearest
//          integer (ties to even) as if the quotient were exact
//   e4m3:  s = 2^e, e the smallest integer >= -126 with a <= 448 * 2^e,
//          code = x / s rounded to the nearest e4m3 value (the division is
//          exact; where code * s would pass the type's largest finite value,
//          the next smaller code)
//
// and a code stands for code * s (float32).  A group that holds an infinity or
// a NaN gets s = NaN, so all of it decodes to NaN: what overflowed in the
// forward pass stays visible in the backward pass.  int8 has one more value that
// does not come back finite: for a = 2^128 - 2^104, the largest float32, s is
// 8454660 * 2^98, and 127 s = 2^128 - 4 * 2^98 rounds to infinity.  (The float32
// below it, 2^128 - 2^105, has s = 8454659 * 2^98 and stays finite.)
//
// int8 is the finer of the two on rows whose groups have no outliers (steps
// of a / 127 against 2^-4 relative), e4m3 keeps small elements next to large
// ones (range 2^18 within a group).
//
// The kernels are HBM-bound, but not by much: some 14 (e4m3) to 20 (int8)
// instructions per element fill the issue slots too, hence the packed maxima
// and float32 pairs below.  A lane owns 16 bytes of input (E elements), a group
// is 16 lanes (16-bit input) or a warp (float32); codes are stored E bytes per
// lane, contiguous over the warp.
#pragma once
#include "esa_f32x2.cuh"

namespace esa {
namespace pack8 {

constexpr int kGroup = 128;
enum Format : int { kInt8 = 0, kE4m3 = 1 };

template <typename T> struct Codes;          // the codes of one 16-byte vector
template <> struct Codes<float> { using Word = uint32_t; };
template <> struct Codes<__nv_bfloat16> { using Word = uint2; };
template <> struct Codes<__half> { using Word = uint2; };

__device__ __forceinline__ uint32_t word_of(const uint32_t& w, int) { return w; }
__device__ __forceinline__ uint32_t word_of(const uint2& w, int i) { return i ? w.y : w.x; }
__device__ __forceinline__ void set_word(uint32_t& w, int, uint32_t v) { w = v; }
__device__ __forceinline__ void set_word(uint2& w, int i, uint32_t v) { (i ? w.y : w.x) = v; }

// Largest magnitude of each of N vectors' groups, as float bits (NaN above
// infinity above finite), on all lanes of the group.  16-bit types compare two
// values per instruction and carry two groups' maxima through one chain of
// shuffles.
template <typename T> struct Max2;
#define ESA_MAX2(T, PTXTYPE)                                                                \
  template <> struct Max2<T> {                                                              \
    __device__ __forceinline__ static uint32_t abs_max(uint32_t a, uint32_t b) {            \
      uint32_t r;                                                                           \
      asm("max.NaN.xorsign.abs." PTXTYPE " %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));        \
      return r;                                                                             \
    }                                                                                       \
  };
ESA_MAX2(__nv_bfloat16, "bf16x2")
ESA_MAX2(__half, "f16x2")
#undef ESA_MAX2

// Float bits of a 16-bit magnitude in the low half of a.
template <typename T> __device__ __forceinline__ uint32_t magnitude_bits(uint32_t a) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return (a & 0x7fffu) << 16;
  return __float_as_uint(__half2float(__ushort_as_half((unsigned short)(a & 0x7fffu))));
}

template <typename T, int N>
__device__ __forceinline__ void group_max(const uint4 (&x)[N], uint32_t (&m)[N]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const uint32_t mask = 0x7fffffffu;
      m[k] = __reduce_max_sync(0xffffffffu, max(max(x[k].x & mask, x[k].y & mask),
                                                max(x[k].z & mask, x[k].w & mask)));
    }
  } else {
    using M = Max2<T>;
#pragma unroll
    for (int k = 0; k < N; k += 2) {
      const uint4 z = make_uint4(0, 0, 0, 0), a = x[k], b = k + 1 < N ? x[k + 1 < N ? k + 1 : k] : z;
      const uint32_t ma = M::abs_max(M::abs_max(a.x, a.y), M::abs_max(a.z, a.w));
      const uint32_t mb = M::abs_max(M::abs_max(b.x, b.y), M::abs_max(b.z, b.w));
      uint32_t r = M::abs_max(__byte_perm(ma, mb, 0x5410), __byte_perm(ma, mb, 0x7632));
#pragma unroll
      for (int o = kGroup / 8 / 2; o > 0; o >>= 1)
        r = M::abs_max(r, __shfl_xor_sync(0xffffffffu, r, o));
      m[k] = magnitude_bits<T>(r);
      if (k + 1 < N) m[k + 1] = magnitude_bits<T>(r >> 16);
    }
  }
}

// Scale of a group with maximum `m` (float bits).
template <int F>
__device__ __forceinline__ float group_scale(uint32_t m) {
  if (m >= 0x7f800000u) return __uint_as_float(0x7fffffffu);
  if constexpr (F == kInt8) {
    // a / 127 correctly rounded: with c the float32 nearest to 1 / 127, one
    // step from q = a c with the exact remainder a - 127 q gives the nearest
    // float32 (Markstein, IBM J. Res. Dev. 34, 1990)
    const float a = __uint_as_float(m), c = 1.f / 127.f;
    const float q = a * c;
    return fmaxf(fmaf(fmaf(-127.f, q, a), c, q), __uint_as_float(0x00800000u));
  } else {
    // m = 1.f * 2^k: e = k - 8, one more when 1.f > 1.75 (448 = 1.75 * 2^8);
    // exponent field of 2^e = field of m - 8 (+ 1), at least 1 (e = -126)
    const int field = (int)(m >> 23) - 8 + ((m & 0x7fffffu) > 0x600000u ? 1 : 0);
    return __uint_as_float((uint32_t)max(field, 1) << 23);
  }
}

// The scale whose code 256 stands for a value above T's largest: 2^8 * 256 =
// 2^16 for fp16, 2^120 * 256 = 2^128 for bf16 and float32.
template <typename T> struct TopScale { static constexpr uint32_t kBits = (120u + 127u) << 23; };
template <> struct TopScale<__half> { static constexpr uint32_t kBits = (8u + 127u) << 23; };

// Codes of E elements of type T with scale s (finite).
template <int F, typename T, int E, typename W>
__device__ __forceinline__ W encode(const float (&x)[E], float s) {
  W out;
  if constexpr (F == kInt8) {
    // x / s within 127 (2^-23 + 2^-24) < 2.3e-5 by the approximate reciprocal;
    // adding 1.5 * 2^23 rounds to an integer, ties to even, and leaves it in
    // the low bits.  Quotients that near to a border between two codes are
    // decided by the remainder, which the fma gives exactly.
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
    constexpr float kMagic = 12582912.f;
    const F2 inv2 = f2(inv, inv), magic = f2(kMagic, kMagic), back = f2(-kMagic, -kMagic);
    uint32_t code[E];
    float off = 0.f;
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      const F2 t = mul2(f2(x[e], x[e + 1]), inv2);
      const F2 r = add2(t, magic);
      const F2 d = fma2(add2(r, back), f2(-1.f, -1.f), t);
      float r0, r1, d0, d1;
      split(r, r0, r1);
      split(d, d0, d1);
      code[e] = __float_as_uint(r0);
      code[e + 1] = __float_as_uint(r1);
      off = fmaxf(off, fmaxf(fabsf(d0), fabsf(d1)));
    }
    if (off > 0.49997f) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float r = __fsub_rn(__uint_as_float(code[e]), kMagic);
        const float d = fmaf(-r, s, x[e]);
        const float ad2 = fabsf(d) + fabsf(d);   // exact, unlike s / 2 next to 2^-126
        if (ad2 > s || (ad2 == s && (code[e] & 1))) code[e] += d > 0.f ? 1u : 0xffffffffu;
      }
    }
#pragma unroll
    for (int e = 0; e < E; e += 4) {
      const uint32_t lo = __byte_perm(code[e], code[e + 1], 0x0040);
      const uint32_t hi = __byte_perm(code[e + 2], code[e + 3], 0x0040);
      set_word(out, e / 4, __byte_perm(lo, hi, 0x5410));
    }
  } else {
    const float inv = __uint_as_float((254u << 23) - __float_as_uint(s));   // 2^-e, exact
    float t[E];
#pragma unroll
    for (int e = 0; e < E; e += 2)
      split(mul2(f2(x[e], x[e + 1]), f2(inv, inv)), t[e], t[e + 1]);
    if (__float_as_uint(s) == TopScale<T>::kBits) {   // 240 is the e4m3 value below 256
#pragma unroll
      for (int e = 0; e < E; ++e) t[e] = fminf(fmaxf(t[e], -240.f), 240.f);
    }
#pragma unroll
    for (int e = 0; e < E; e += 4) {
      uint32_t w;
      asm("{\n\t.reg .b16 lo, hi;\n\t"
          "cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\t"
          "cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\t"
          "mov.b32 %0, {lo, hi};\n\t}"
          : "=r"(w)
          : "f"(t[e]), "f"(t[e + 1]), "f"(t[e + 2]), "f"(t[e + 3]));
      set_word(out, e / 4, w);
    }
  }
  return out;
}

// The values that E codes with scale s stand for.
template <int F, int E, typename W>
__device__ __forceinline__ void decode(const W& c, float s, float (&x)[E]) {
  const F2 s2 = f2(s, s);
#pragma unroll
  for (int e = 0; e < E; e += 4) {
    const uint32_t w = word_of(c, e / 4);
    F2 lo, hi;
    if constexpr (F == kInt8) {
      // code + 128 into the low mantissa bits of 2^23, then subtract 2^23 + 128
      const uint32_t u = w ^ 0x80808080u;
      const F2 bias = f2(-8388736.f, -8388736.f);
      float b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) b[i] = __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7440 + i));
      lo = add2(f2(b[0], b[1]), bias);
      hi = add2(f2(b[2], b[3]), bias);
    } else {
      uint32_t a, b;
      asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\t"
          "cvt.rn.f16x2.e4m3x2 %0, lo;\n\tcvt.rn.f16x2.e4m3x2 %1, hi;\n\t}"
          : "=r"(a), "=r"(b)
          : "r"(w));
      const float2 p = __half22float2(*reinterpret_cast<__half2*>(&a));
      const float2 q = __half22float2(*reinterpret_cast<__half2*>(&b));
      lo = f2(p.x, p.y);
      hi = f2(q.x, q.y);
    }
    split(mul2(lo, s2), x[e], x[e + 1]);
    split(mul2(hi, s2), x[e + 2], x[e + 3]);
  }
}

// Codes of one lane's vector of a group with maximum m, stored with, from the
// group's first lane, the scale.
template <int F, typename T, int E>
__device__ __forceinline__ void pack_vec(const float (&x)[E], uint32_t m, uint8_t* code_dst,
                                         float* scale_dst) {
  using W = typename Codes<T>::Word;
  const float s = group_scale<F>(m);
  W c{};
  if (m < 0x7f800000u) c = encode<F, T, E, W>(x, s);
  *reinterpret_cast<W*>(code_dst) = c;
  if ((threadIdx.x & (kGroup / E - 1)) == 0) *scale_dst = s;
}

// ---------------------------------------------------------------------------
// Rows to codes and back.  A warp takes K * 32 consecutive vectors of one row
// and issues all their loads first.  The grid covers the rows once: CTAs that
// stride over them leave SMs idle at the end.
// ---------------------------------------------------------------------------
constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
// K by kernel, measured at 16384 x 22016 bf16 (int8 / e4m3): quantize 203 / 159
// us (K = 2: 231 / 167), SwiGLU forward 265 / 221 (K = 2: 279 / 234), SwiGLU
// backward 267 / 266 (K = 4: 268 / 270).  HBM's times are 167, 222 and 277.
constexpr int kRowUnits = 4;         // quantize, dequantize
constexpr int kSwigluFwdUnits = 4;
constexpr int kSwigluBwdUnits = 2;

// This warp's part of a row; rows * parts per row is below 2^32.
template <int K>
struct Part {
  int64_t row;
  int vec;                     // this lane's first vector; the others are 32 apart
  int vpr;                     // vectors per row
  __device__ __forceinline__ Part(int vecs_per_row) : vpr(vecs_per_row) {
    const uint32_t parts = (vpr + 32 * K - 1) / (32 * K);
    const uint32_t task = blockIdx.x * kWarps + (threadIdx.x >> 5);
    const uint32_t r = task / parts;
    row = r;
    vec = (task - r * parts) * (32 * K) + (threadIdx.x & 31);
  }
  __device__ __forceinline__ bool in(int k) const { return vec + k * 32 < vpr; }
};

template <typename T, int F>
__global__ void __launch_bounds__(kThreads)
quantize_kernel(int64_t rows, int dim, const T* __restrict__ x, uint8_t* __restrict__ codes,
                float* __restrict__ scales) {
  using V = Vec<T>;
  constexpr int E = V::kElems, K = kRowUnits;
  const Part<K> u(dim / E);
  if (u.row >= rows) return;
  const int64_t at = u.row * dim + u.vec * E;
  uint4 raw[K];
#pragma unroll
  for (int k = 0; k < K; ++k)
    raw[k] = u.in(k) ? ldg16_stream(x + at + k * 32 * E) : make_uint4(0, 0, 0, 0);
  uint32_t m[K];
  group_max<T, K>(raw, m);
  float* scale = scales + u.row * ((dim + kGroup - 1) / kGroup) + u.vec * E / kGroup;
#pragma unroll
  for (int k = 0; k < K; ++k)
    if (u.in(k)) {
      float f[E];
      V::to_float(raw[k], f);
      pack_vec<F, T>(f, m[k], codes + at + k * 32 * E, scale + k * 32 * E / kGroup);
    }
}

template <typename T, int F>
__global__ void __launch_bounds__(kThreads)
dequantize_kernel(int64_t rows, int dim, const uint8_t* __restrict__ codes,
                  const float* __restrict__ scales, T* __restrict__ x) {
  using V = Vec<T>;
  using W = typename Codes<T>::Word;
  constexpr int E = V::kElems, K = kRowUnits;
  const Part<K> u(dim / E);
  if (u.row >= rows) return;
  const int64_t at = u.row * dim + u.vec * E;
  const float* scale = scales + u.row * ((dim + kGroup - 1) / kGroup) + u.vec * E / kGroup;
  W c[K];
  float s[K];
#pragma unroll
  for (int k = 0; k < K; ++k)
    if (u.in(k)) {
      c[k] = *reinterpret_cast<const W*>(codes + at + k * 32 * E);
      s[k] = __ldg(scale + k * 32 * E / kGroup);
    }
#pragma unroll
  for (int k = 0; k < K; ++k)
    if (u.in(k)) {
      float f[E];
      decode<F, E>(c[k], s[k], f);
      stg16(x + at + k * 32 * E, V::from_float(f));
    }
}

// ---------------------------------------------------------------------------
// RMSNorm (with an optional residual add) that also writes h in 8 bits, and
// its counterpart in the backward pass: h from the codes, normalised again.
// W warps own a row and keep it in registers, NV <= 4 vectors per lane: all of
// a row's loads are issued before the first is used, and 4 vectors leave room
// for enough rows per SM to keep HBM busy while others are summed.
// ---------------------------------------------------------------------------
template <int W> constexpr int kNormThreads = W > 4 ? 32 * W : 128;
template <int W> constexpr int kNormRows = kNormThreads<W> / (32 * W);   // rows per CTA

// Sum of v over the W warps of a row; red has a float per warp of the CTA.
template <int W>
__device__ __forceinline__ float row_total(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if constexpr (W > 1) {
    const int warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) red[warp] = v;
    __syncthreads();
    const int w0 = warp / W * W;
    v = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) v += red[w0 + w];
  }
  return v;
}

// h (already rounded to T) -> y of this lane's vectors.
template <typename T, int NV, int W>
__device__ __forceinline__ void norm_vecs(const uint4 (&h)[NV], int vpr, int vec0, float rs,
                                          const T* __restrict__ w, T* y) {
  using V = Vec<T>;
  constexpr int E = V::kElems;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int vec = vec0 + j * W * 32;
    if (vec < vpr) {
      float f[E], wv[E];
      V::to_float(h[j], f);
      V::to_float(ldg16(w + vec * E), wv);
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] = f[e] * rs * wv[e];
      stg16(y + vec * E, V::from_float(f));
    }
  }
}

template <typename T, int F, int NV, int W>
__global__ void __launch_bounds__(kNormThreads<W>)
norm_pack_kernel(int64_t rows, int dim, const T* __restrict__ x, const T* __restrict__ res,
                 T* __restrict__ h_out, const T* __restrict__ w, float eps, T* __restrict__ y,
                 float* __restrict__ rstd, uint8_t* __restrict__ codes,
                 float* __restrict__ scales) {
  using V = Vec<T>;
  constexpr int E = V::kElems;
  __shared__ float red[kNormThreads<W> / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int groups = (dim + kGroup - 1) / kGroup;
  const int64_t row = (int64_t)blockIdx.x * kNormRows<W> + warp / W;
  const int vpr = row < rows ? dim / E : 0;        // no vectors past the last row
  const int vec0 = (warp % W) * 32 + lane;
  const int64_t at = row * dim;
  uint4 h[NV], r[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int vec = vec0 + j * W * 32;
    h[j] = vec < vpr ? ldg16_stream(x + at + vec * E) : make_uint4(0, 0, 0, 0);
    r[j] = res && vec < vpr ? ldg16_stream(res + at + vec * E) : make_uint4(0, 0, 0, 0);
  }
  if (res) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int vec = vec0 + j * W * 32;
      float f[E], rf[E];
      V::to_float(h[j], f);
      V::to_float(r[j], rf);
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] += rf[e];
      h[j] = V::from_float(f);   // the stored h is what is normed and packed
      if (vec < vpr) stg16(h_out + at + vec * E, h[j]);
    }
  }
  uint32_t m[NV];
  group_max<T, NV>(h, m);
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int vec = vec0 + j * W * 32;
    float f[E];
    V::to_float(h[j], f);
#pragma unroll
    for (int e = 0; e < E; ++e) ss = fmaf(f[e], f[e], ss);
    if (vec < vpr)
      pack_vec<F, T>(f, m[j], codes + at + vec * E, scales + row * groups + vec * E / kGroup);
  }
  const float rs = rsqrtf(row_total<W>(ss, red) / (float)dim + eps);
  norm_vecs<T, NV, W>(h, vpr, vec0, rs, w, y + at);
  if (vec0 == 0 && vpr) rstd[row] = rs;
}

template <typename T, int F, int NV, int W>
__global__ void __launch_bounds__(kNormThreads<W>)
unpack_norm_kernel(int64_t rows, int dim, const uint8_t* __restrict__ codes,
                   const float* __restrict__ scales, T* __restrict__ h_out,
                   const T* __restrict__ w, float eps, T* __restrict__ y,
                   float* __restrict__ rstd) {
  using V = Vec<T>;
  using C = typename Codes<T>::Word;
  constexpr int E = V::kElems;
  __shared__ float red[kNormThreads<W> / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int groups = (dim + kGroup - 1) / kGroup;
  const int64_t row = (int64_t)blockIdx.x * kNormRows<W> + warp / W;
  const int vpr = row < rows ? dim / E : 0;
  const int vec0 = (warp % W) * 32 + lane;
  const int64_t at = row * dim;
  C c[NV];
  float s[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int vec = vec0 + j * W * 32;
    c[j] = C{};
    s[j] = 0.f;
    if (vec < vpr) {
      c[j] = *reinterpret_cast<const C*>(codes + at + vec * E);
      s[j] = __ldg(scales + row * groups + vec * E / kGroup);
    }
  }
  uint4 h[NV];
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int vec = vec0 + j * W * 32;
    float f[E];
    decode<F, E>(c[j], s[j], f);
    h[j] = V::from_float(f);
    if (vec < vpr) stg16(h_out + at + vec * E, h[j]);
    V::to_float(h[j], f);
#pragma unroll
    for (int e = 0; e < E; ++e) ss = fmaf(f[e], f[e], ss);
  }
  const float rs = rsqrtf(row_total<W>(ss, red) / (float)dim + eps);
  norm_vecs<T, NV, W>(h, vpr, vec0, rs, w, y + at);
  if (vec0 == 0 && vpr) rstd[row] = rs;
}

// ---------------------------------------------------------------------------
// SwiGLU that also writes its gate / up rows in 8 bits (two rows of ffn
// elements per token, each with its own groups), and its backward from them.
// ---------------------------------------------------------------------------
// s = sigmoid(g) and c = 1 - s from e = exp(-|g|) <= 1, so that neither
// overflows nor cancels.  16-bit types take the hardware's exp2 and reciprocal
// (relative error below 2^-22 + |g| 2^-24, far inside their rounding), float32
// expf and a division: those in every type cost 50 of 330 us (16384 x 11008
// bf16, forward).
template <typename T>
__device__ __forceinline__ void sigmoid_of(float g, float& s, float& c) {
  float e, r;
  if constexpr (sizeof(T) == 4) {
    e = expf(-fabsf(g));
    r = 1.f / (1.f + e);
  } else {
    e = __expf(-fabsf(g));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));   // of [1, 2]
  }
  const float er = e * r;
  s = g >= 0.f ? r : er;
  c = g >= 0.f ? er : r;
}

template <typename T, int F>
__global__ void __launch_bounds__(kThreads)
swiglu_pack_kernel(int64_t rows, int ffn, const T* __restrict__ gu, T* __restrict__ out,
                   uint8_t* __restrict__ codes, float* __restrict__ scales) {
  using V = Vec<T>;
  constexpr int E = V::kElems, K = kSwigluFwdUnits;
  const Part<K> u(ffn / E);
  if (u.row >= rows) return;
  const int groups = (ffn + kGroup - 1) / kGroup;
  const int64_t at = u.row * 2 * ffn + u.vec * E;
  uint4 raw[2 * K];               // gate and up vectors in turn
#pragma unroll
  for (int k = 0; k < K; ++k) {
    raw[2 * k] = raw[2 * k + 1] = make_uint4(0, 0, 0, 0);
    if (u.in(k)) {
      raw[2 * k] = ldg16_stream(gu + at + k * 32 * E);
      raw[2 * k + 1] = ldg16_stream(gu + at + ffn + k * 32 * E);
    }
  }
  uint32_t m[2 * K];
  group_max<T, 2 * K>(raw, m);
  uint8_t* code = codes + at;
  float* scale = scales + u.row * 2 * groups + u.vec * E / kGroup;
  T* dst = out + u.row * ffn + u.vec * E;
#pragma unroll
  for (int k = 0; k < K; ++k)
    if (u.in(k)) {
      float g[E], up[E], o[E];
      V::to_float(raw[2 * k], g);
      V::to_float(raw[2 * k + 1], up);
      pack_vec<F, T>(g, m[2 * k], code + k * 32 * E, scale + k * 32 * E / kGroup);
      pack_vec<F, T>(up, m[2 * k + 1], code + ffn + k * 32 * E,
                     scale + groups + k * 32 * E / kGroup);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float s, c;
        sigmoid_of<T>(g[e], s, c);
        o[e] = g[e] * s * up[e];
      }
      stg16(dst + k * 32 * E, V::from_float(o));
    }
}

template <typename T, int F>
__global__ void __launch_bounds__(kThreads)
swiglu_unpack_bwd_kernel(int64_t rows, int ffn, const uint8_t* __restrict__ codes,
                         const float* __restrict__ scales, const T* __restrict__ dout,
                         T* __restrict__ dgu, T* __restrict__ out_re) {
  using V = Vec<T>;
  using W = typename Codes<T>::Word;
  constexpr int E = V::kElems, K = kSwigluBwdUnits;
  const Part<K> u(ffn / E);
  if (u.row >= rows) return;
  const int groups = (ffn + kGroup - 1) / kGroup;
  const int64_t at = u.row * 2 * ffn + u.vec * E, at1 = u.row * ffn + u.vec * E;
  const float* scale = scales + u.row * 2 * groups + u.vec * E / kGroup;
  W cg[K], cu[K];
  float sg[K], su[K];
  uint4 raw_d[K];
#pragma unroll
  for (int k = 0; k < K; ++k)
    if (u.in(k)) {
      cg[k] = *reinterpret_cast<const W*>(codes + at + k * 32 * E);
      cu[k] = *reinterpret_cast<const W*>(codes + at + ffn + k * 32 * E);
      sg[k] = __ldg(scale + k * 32 * E / kGroup);
      su[k] = __ldg(scale + groups + k * 32 * E / kGroup);
      raw_d[k] = ldg16_stream(dout + at1 + k * 32 * E);
    }
#pragma unroll
  for (int k = 0; k < K; ++k)
    if (u.in(k)) {
      float g[E], up[E], d[E], dg[E], du[E], o[E];
      decode<F, E>(cg[k], sg[k], g);
      decode<F, E>(cu[k], su[k], up);
      V::to_float(raw_d[k], d);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float s, c;
        sigmoid_of<T>(g[e], s, c);
        const float silu = g[e] * s;
        dg[e] = d[e] * up[e] * fmaf(silu, c, s);        // s (1 + g (1 - s))
        du[e] = d[e] * silu;
        o[e] = silu * up[e];
      }
      stg16(dgu + at + k * 32 * E, V::from_float(dg));
      stg16(dgu + at + ffn + k * 32 * E, V::from_float(du));
      if (out_re) stg16(out_re + at1 + k * 32 * E, V::from_float(o));
    }
}

}  // namespace pack8
}  // namespace esa
