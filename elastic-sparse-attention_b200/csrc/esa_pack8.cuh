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
// forward pass stays visible in the backward pass.
//
// int8 is the finer of the two on rows whose groups have no outliers (steps
// of a / 127 against 2^-4 relative), e4m3 keeps small elements next to large
// ones (range 2^18 within a group).
//
// The kernels are HBM-bound.  A lane owns 16 bytes of input (E elements), a
// group is 16 lanes (16-bit input) or a warp (float32): its maximum is a few
// shuffles, and codes are stored E bytes per lane, contiguous over the warp.
#pragma once
#include "esa_common.cuh"

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

// Largest |x| of the group as float bits (NaN above infinity above finite);
// all lanes of the group return it.
template <int E>
__device__ __forceinline__ uint32_t group_max(const float (&x)[E]) {
  float a = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e)      // the maximum of the hardware, with NaN passed on
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(fabsf(x[e])));
  uint32_t m = __float_as_uint(a) & 0x7fffffffu;
#pragma unroll
  for (int o = kGroup / E / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}

// Scale of a group with maximum `m` (float bits).
template <int F>
__device__ __forceinline__ float group_scale(uint32_t m) {
  if (m >= 0x7f800000u) return __uint_as_float(0x7fffffffu);
  if constexpr (F == kInt8) {
    return fmaxf(__fdiv_rn(__uint_as_float(m), 127.f), __uint_as_float(0x00800000u));
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
    // x / s within 2^-16 by the reciprocal; adding 1.5 * 2^23 rounds to an
    // integer, ties to even, and leaves it in the low bits.  Quotients that
    // near to a border between two codes are decided by the remainder, which
    // the fma gives exactly.
    const float inv = __frcp_rn(s);
    constexpr float kMagic = 12582912.f;
    uint32_t code[E];
    float off = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float t = x[e] * inv;
      const float r = __fadd_rn(t, kMagic);
      code[e] = __float_as_uint(r);
      off = fmaxf(off, fabsf(__fsub_rn(t, __fsub_rn(r, kMagic))));
    }
    if (off > 0.4999f) {
      const float half = 0.5f * s;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float r = __fsub_rn(__uint_as_float(code[e]), kMagic);
        const float d = fmaf(-r, s, x[e]);
        const float ad = fabsf(d);
        if (ad > half || (ad == half && (code[e] & 1))) code[e] += d > 0.f ? 1u : 0xffffffffu;
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
    for (int e = 0; e < E; ++e) t[e] = x[e] * inv;
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
#pragma unroll
  for (int e = 0; e < E; e += 4) {
    const uint32_t w = word_of(c, e / 4);
    if constexpr (F == kInt8) {
      // code + 128 into the low mantissa bits of 2^23, then subtract 2^23 + 128
      const uint32_t u = w ^ 0x80808080u;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        x[e + i] = __fsub_rn(__uint_as_float(__byte_perm(u, 0x4B000000u, 0x7440 + i)),
                             8388736.f) * s;
    } else {
      uint32_t a, b;
      asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\t"
          "cvt.rn.f16x2.e4m3x2 %0, lo;\n\tcvt.rn.f16x2.e4m3x2 %1, hi;\n\t}"
          : "=r"(a), "=r"(b)
          : "r"(w));
      float2 f = __half22float2(*reinterpret_cast<__half2*>(&a));
      x[e] = f.x * s;
      x[e + 1] = f.y * s;
      f = __half22float2(*reinterpret_cast<__half2*>(&b));
      x[e + 2] = f.x * s;
      x[e + 3] = f.y * s;
    }
  }
}

// Encodes one lane's vector (all lanes of the warp call it; lanes past the
// row's end pass in = false and zeros) and stores the codes and, from the
// group's first lane, the scale.
template <int F, typename T, int E>
__device__ __forceinline__ void pack_vec(const float (&x)[E], bool in, uint8_t* code_dst,
                                         float* scale_dst) {
  using W = typename Codes<T>::Word;
  const uint32_t m = group_max<E>(x);
  const float s = group_scale<F>(m);
  if (!in) return;
  W c;
  if (m >= 0x7f800000u) {
#pragma unroll
    for (int i = 0; i < E / 4; ++i) set_word(c, i, 0u);
  } else {
    c = encode<F, T, E, W>(x, s);
  }
  *reinterpret_cast<W*>(code_dst) = c;
  if ((threadIdx.x & (kGroup / E - 1)) == 0) *scale_dst = s;
}

// ---------------------------------------------------------------------------
// Rows to codes and back.  A warp's unit is 32 vectors of one row.
// ---------------------------------------------------------------------------
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

template <typename T, int F>
__global__ void __launch_bounds__(kThreads)
quantize_kernel(int64_t rows, int dim, const T* __restrict__ x, uint8_t* __restrict__ codes,
                float* __restrict__ scales) {
  using V = Vec<T>;
  constexpr int E = V::kElems;
  const int lane = threadIdx.x & 31;
  const int vpr = dim / E, upr = (vpr + 31) / 32, groups = (dim + kGroup - 1) / kGroup;
  const int64_t units = rows * upr;
  for (int64_t u = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5); u < units;
       u += (int64_t)gridDim.x * kWarps) {
    const int64_t row = u / upr;
    const int vec = (int)(u - row * upr) * 32 + lane;
    const bool in = vec < vpr;
    float f[E] = {};
    if (in) V::to_float(ldg16_stream(x + row * dim + (int64_t)vec * E), f);
    pack_vec<F, T>(f, in, codes + row * dim + (int64_t)vec * E,
                   scales + row * groups + vec * E / kGroup);
  }
}

template <typename T, int F>
__global__ void __launch_bounds__(kThreads)
dequantize_kernel(int64_t rows, int dim, const uint8_t* __restrict__ codes,
                  const float* __restrict__ scales, T* __restrict__ x) {
  using V = Vec<T>;
  using W = typename Codes<T>::Word;
  constexpr int E = V::kElems;
  const int lane = threadIdx.x & 31;
  const int vpr = dim / E, upr = (vpr + 31) / 32, groups = (dim + kGroup - 1) / kGroup;
  const int64_t units = rows * upr;
  for (int64_t u = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5); u < units;
       u += (int64_t)gridDim.x * kWarps) {
    const int64_t row = u / upr;
    const int vec = (int)(u - row * upr) * 32 + lane;
    if (vec >= vpr) continue;
    float f[E];
    decode<F, E>(*reinterpret_cast<const W*>(codes + row * dim + (int64_t)vec * E),
                 __ldg(scales + row * groups + vec * E / kGroup), f);
    stg16(x + row * dim + (int64_t)vec * E, V::from_float(f));
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
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int vec = vec0 + j * W * 32;
    const bool in = vec < vpr;
    float f[E];
    V::to_float(h[j], f);
    if (res) {
      float rf[E];
      V::to_float(r[j], rf);
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] += rf[e];
      h[j] = V::from_float(f);   // the stored h is what is normed and packed
      if (in) stg16(h_out + at + vec * E, h[j]);
      V::to_float(h[j], f);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) ss = fmaf(f[e], f[e], ss);
    if (vec - lane < vpr)        // the warp's 32 vectors begin inside the row
      pack_vec<F, T>(f, in, codes + at + vec * E, scales + row * groups + vec * E / kGroup);
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
// expf and a division: with these in every type the kernels are bound by
// instructions (16384 x 11008 bf16: 329 us forward instead of HBM's 222).
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
  constexpr int E = V::kElems;
  const int lane = threadIdx.x & 31;
  const int vpr = ffn / E, upr = (vpr + 31) / 32, groups = (ffn + kGroup - 1) / kGroup;
  const int64_t units = rows * upr;
  for (int64_t u = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5); u < units;
       u += (int64_t)gridDim.x * kWarps) {
    const int64_t row = u / upr;
    const int vec = (int)(u - row * upr) * 32 + lane;
    const bool in = vec < vpr;
    const int64_t at = row * 2 * ffn + (int64_t)vec * E;
    float g[E] = {}, up[E] = {};
    if (in) {
      V::to_float(ldg16_stream(gu + at), g);
      V::to_float(ldg16_stream(gu + at + ffn), up);
    }
    const int64_t sc = row * 2 * groups + vec * E / kGroup;
    pack_vec<F, T>(g, in, codes + at, scales + sc);
    pack_vec<F, T>(up, in, codes + at + ffn, scales + sc + groups);
    if (in) {
      float o[E];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float s, c;
        sigmoid_of<T>(g[e], s, c);
        o[e] = g[e] * s * up[e];
      }
      stg16(out + row * ffn + (int64_t)vec * E, V::from_float(o));
    }
  }
}

template <typename T, int F>
__global__ void __launch_bounds__(kThreads)
swiglu_unpack_bwd_kernel(int64_t rows, int ffn, const uint8_t* __restrict__ codes,
                         const float* __restrict__ scales, const T* __restrict__ dout,
                         T* __restrict__ dgu, T* __restrict__ out_re) {
  using V = Vec<T>;
  using W = typename Codes<T>::Word;
  constexpr int E = V::kElems;
  const int lane = threadIdx.x & 31;
  const int vpr = ffn / E, upr = (vpr + 31) / 32, groups = (ffn + kGroup - 1) / kGroup;
  const int64_t units = rows * upr;
  for (int64_t u = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5); u < units;
       u += (int64_t)gridDim.x * kWarps) {
    const int64_t row = u / upr;
    const int vec = (int)(u - row * upr) * 32 + lane;
    if (vec >= vpr) continue;
    const int64_t at = row * 2 * ffn + (int64_t)vec * E;
    const int64_t sc = row * 2 * groups + vec * E / kGroup;
    float g[E], up[E], d[E], dg[E], du[E], o[E];
    decode<F, E>(*reinterpret_cast<const W*>(codes + at), __ldg(scales + sc), g);
    decode<F, E>(*reinterpret_cast<const W*>(codes + at + ffn), __ldg(scales + sc + groups), up);
    V::to_float(ldg16_stream(dout + row * ffn + (int64_t)vec * E), d);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      float s, c;
      sigmoid_of<T>(g[e], s, c);
      const float silu = g[e] * s;
      dg[e] = d[e] * up[e] * fmaf(silu, c, s);        // s (1 + g (1 - s))
      du[e] = d[e] * silu;
      o[e] = silu * up[e];
    }
    stg16(dgu + at, V::from_float(dg));
    stg16(dgu + at + ffn, V::from_float(du));
    if (out_re) stg16(out_re + row * ffn + (int64_t)vec * E, V::from_float(o));
  }
}

}  // namespace pack8
}  // namespace esa
