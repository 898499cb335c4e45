// Keys and values cached in 4 bits (esa_int4.cuh, groups of 32 along the head
// dimension) and the elastic attention that reads them.
//
// A cached row of one K/V head is D / 2 bytes of key codes, D / 2 bytes of value
// codes (one 128-byte line for D = 128) and 2 x D / 32 bf16 scales.  The codes
// lie in the order in which the matrix instructions take them:
//   key:   word t * (D / 32) + c of a row (t < 4, c < D / 32) holds the elements
//          c * 32 + t * 8 + i, nibble i
//   value: word g * (D / 64) + c (g < 8, c < D / 64) holds the elements
//          c * 64 + i * 8 + g, nibble i
//
// Attention: every (query row, head) pair has w keys of its own, so nothing is
// shared between pairs and the work is decoding 2 w D codes.  The products run
// on mma.sync m16n8k16 (f16, float32 sums) with the codes as A and the query,
// or the weights, in the columns of B that one vector leaves free otherwise:
//   scores: A = 16 keys x 16 elements, B column = the query in f16 (its float32
//           form in three parts), per group of 32 a sum of its own, times the scale
//   output: A = 16 elements x 16 keys, B column = (group, part) with the weight
//           times that group's scale in two or three f16 parts; an output element
//           reads the columns of its group
// A code is used as the f16 denormal that its nibble is (n 2^-24, or n 2^-20 one
// nibble up, taken back in B or in the result), so decoding costs one AND per two
// codes and no conversion; what the stored + 8 adds is 8 times the sum of the
// column, formed by one product with a matrix of ones.  Queries and weights are
// scaled by a power of two to just below 2^15 before they are cut to f16: 22 bits
// (two parts) or 33 (three) below the largest.
//
// A warp takes 32 slots of a pair at a time, all their loads in flight, with an
// online softmax in float32; with few pairs a pair's slots are split over the
// warps of a CTA and joined in shared memory.
#pragma once
#include "esa_int4.cuh"

namespace esa {
namespace cache4 {

constexpr int kGroup = 32;
constexpr int kErrKvRange = 1, kErrQueryRange = 4;     // ESA_DEVERR_KV_RANGE, _QUERY_RANGE

struct Cache {
  uint8_t* codes;             // [B, Hkv, S, 2, D / 2]
  __nv_bfloat16* scales;      // [B, Hkv, S, 2, D / 32]
  int B, Hkv;
  int64_t S;
};

// Rows of a call: row l < count(b) of sequence b is position start(b) + l.
struct Span {
  const int64_t* start;       // [B] or null: start0 for all
  const int64_t* counts;      // [B] or null: all rows
  int64_t start0, L;
  __device__ __forceinline__ int64_t begin(int b) const { return start ? start[b] : start0; }
  __device__ __forceinline__ int64_t count(int b) const {
    if (!counts) return L;
    const int64_t c = counts[b];
    return c < 0 ? 0 : c < L ? c : L;
  }
  // Position of row l of sequence b; -1 padding, -2 outside the cache.
  __device__ __forceinline__ int64_t position(int b, int64_t l, int64_t S) const {
    if (l >= count(b)) return -1;
    const int64_t s = begin(b);
    return s < 0 || s >= S - l ? -2 : s + l;
  }
};

// 8 lanes with 8 nibbles each: nibble i of lane j <-> nibble j of lane i.
__device__ __forceinline__ uint32_t transpose8(uint32_t w, int j) {
  uint32_t o = __shfl_xor_sync(0xffffffffu, w, 4);
  w = j & 4 ? (w & 0xffff0000u) | (o >> 16) : (w & 0x0000ffffu) | (o << 16);
  o = __shfl_xor_sync(0xffffffffu, w, 2);
  w = j & 2 ? (w & 0xff00ff00u) | ((o >> 8) & 0x00ff00ffu) : (w & 0x00ff00ffu) | ((o << 8) & 0xff00ff00u);
  o = __shfl_xor_sync(0xffffffffu, w, 1);
  return j & 1 ? (w & 0xf0f0f0f0u) | ((o >> 4) & 0x0f0f0f0fu) : (w & 0x0f0f0f0fu) | ((o << 4) & 0xf0f0f0f0u);
}

// ---------------------------------------------------------------------------
// Rows into the cache and out of it.  A thread owns 8 elements of a head row (of
// k and of v); D / 8 neighbouring threads a row; rows in the order [B, L, H], as a
// projection leaves them.
// ---------------------------------------------------------------------------
struct Heads { const void* data; int64_t sb, sh, ss; };

constexpr int kRowThreads = 256;

template <typename T> struct RowParams {
  Cache c;
  Span span;
  Heads k, v;
  int64_t units;              // B * L * Hkv * D / 8
  int* err;
};

template <int D> struct Unit {          // which 8 elements a thread owns
  int64_t l;
  int b, h, part;
  template <typename T>
  __device__ __forceinline__ Unit(const RowParams<T>& p, int64_t u) {
    constexpr int PER = D / 8;
    part = (int)(u % PER);
    const int64_t r = u / PER, bl = r / p.c.Hkv;
    h = (int)(r % p.c.Hkv);
    b = (int)(bl / p.span.L);
    l = bl % p.span.L;
  }
  __device__ __forceinline__ int key_word() const { return (part & 3) * (D / 32) + (part >> 2); }
  __device__ __forceinline__ int value_word() const { return (part & 7) * (D / 64) + (part >> 3); }
};

// Codes (one nibble each) and scale of 8 elements whose group is 4 neighbouring lanes.
__device__ __forceinline__ uint32_t encode8(const float (&f)[8], float& s) {
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, int4::abs_bits(f[e]));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
  s = int4::group_scale(top);
  const float inv = 1.f / s;
  uint32_t w = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) w |= int4::code_of(f[e], s, inv) << (4 * e);
  return w;
}

template <typename T>
__device__ __forceinline__ void load8(const Heads& h, int b, int head, int64_t l, int part, bool in,
                                      float (&f)[8]) {
  const T* p = static_cast<const T*>(h.data) + b * h.sb + head * h.sh + l * h.ss + part * 8;
#pragma unroll
  for (int i = 0; i < 8 / Vec<T>::kElems; ++i) {
    const uint4 v = in ? ldg16_stream(p + i * Vec<T>::kElems) : make_uint4(0, 0, 0, 0);
    Vec<T>::to_float(v, f + i * Vec<T>::kElems);
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kRowThreads)
write_kernel(const RowParams<T> p) {
  const int64_t u = (int64_t)blockIdx.x * kRowThreads + threadIdx.x;
  const bool in = u < p.units;
  const Unit<D> e(p, in ? u : p.units - 1);
  int64_t pos = p.span.position(e.b, e.l, p.c.S);
  if (pos == -2 && in && p.err) atomicOr(p.err, kErrKvRange);
  const bool go = in && pos >= 0;
  float f[8], sk, sv;
  load8<T>(p.k, e.b, e.h, e.l, e.part, go, f);
  const uint32_t kw = encode8(f, sk);
  load8<T>(p.v, e.b, e.h, e.l, e.part, go, f);
  const uint32_t vw = transpose8(encode8(f, sv), e.part & 7);
  if (!go) return;
  const int64_t row = ((int64_t)e.b * p.c.Hkv + e.h) * p.c.S + pos;
  uint32_t* codes = reinterpret_cast<uint32_t*>(p.c.codes + row * D);
  codes[e.key_word()] = kw;
  codes[D / 8 + e.value_word()] = vw;
  if ((e.part & 3) == 0) {
    __nv_bfloat16* s = p.c.scales + row * (2 * D / kGroup) + (e.part >> 2);
    s[0] = __float2bfloat16_rn(sk);
    s[D / kGroup] = __float2bfloat16_rn(sv);
  }
}

template <typename T>
__device__ __forceinline__ void store8(const Heads& h, int b, int head, int64_t l, int part,
                                       uint32_t w, float s) {
  T* p = static_cast<T*>(const_cast<void*>(h.data)) + b * h.sb + head * h.sh + l * h.ss + part * 8;
  float f[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = int4::decode(w >> (4 * e), s);
#pragma unroll
  for (int i = 0; i < 8 / Vec<T>::kElems; ++i)
    stg16(p + i * Vec<T>::kElems, Vec<T>::from_float(f + i * Vec<T>::kElems));
}

// Rows outside the cache come out as zeros.
template <typename T, int D>
__global__ void __launch_bounds__(kRowThreads)
read_kernel(const RowParams<T> p) {
  const int64_t u = (int64_t)blockIdx.x * kRowThreads + threadIdx.x;
  const bool in = u < p.units;
  const Unit<D> e(p, in ? u : p.units - 1);
  const int64_t pos = p.span.position(e.b, e.l, p.c.S);
  const bool go = in && pos >= 0;
  if (pos == -2 && in && p.err) atomicOr(p.err, kErrKvRange);
  uint32_t kw = 0x88888888u, vw = kw;
  float sk = 0.f, sv = 0.f;
  if (go) {
    const int64_t row = ((int64_t)e.b * p.c.Hkv + e.h) * p.c.S + pos;
    const uint32_t* codes = reinterpret_cast<const uint32_t*>(p.c.codes + row * D);
    kw = __ldg(codes + e.key_word());
    vw = __ldg(codes + D / 8 + e.value_word());
    const __nv_bfloat16* s = p.c.scales + row * (2 * D / kGroup) + (e.part >> 2);
    sk = __bfloat162float(s[0]);
    sv = __bfloat162float(s[D / kGroup]);
  }
  vw = transpose8(vw, e.part & 7);
  if (!in) return;
  store8<T>(p.k, e.b, e.h, e.l, e.part, kw, sk);
  store8<T>(p.v, e.b, e.h, e.l, e.part, vw, sv);
}

// ---------------------------------------------------------------------------
// Attention.
// ---------------------------------------------------------------------------
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                    uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 2^e with x 2^e in [2^14, 2^15) for the float bits of x >= 0 (x = 0, or too
// small for that: 2^126), and its inverse.
__device__ __forceinline__ float lift(uint32_t bits, float& inverse) {
  const int field = min(253, 14 + 254 - (int)(bits >> 23));
  inverse = __uint_as_float((uint32_t)(254 - field) << 23);
  return __uint_as_float((uint32_t)field << 23);
}

__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Part `part` of (lo, hi) in f16: what the parts before it leave, rounded.
template <int PARTS>
__device__ __forceinline__ uint32_t half_part(float lo, float hi, int part) {
  uint32_t h = half2_bits(lo, hi);
#pragma unroll
  for (int i = 1; i < PARTS; ++i) {
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&h));
    if (part >= i) {
      lo -= v.x;
      hi -= v.y;
      h = half2_bits(lo, hi);
    }
  }
  return part < PARTS ? h : 0u;
}

template <typename T> struct AttendParams {
  Cache c;
  Span span;
  Heads q, o;
  int Hq, G;                  // query heads, query heads per K/V head
  int64_t pairs;              // B * L * Hq
  int warps_per_pair;         // 1, 2, 4 or 8
  Pattern pat;
  float scale_log2;
  float* lse;                 // [B, Hq, L]
  int* err;
};

constexpr int kAttendWarps = 8;

template <int N> __device__ __forceinline__ void load_words(const void* at, bool in, uint32_t (&w)[N]) {
  const uint32_t* p = static_cast<const uint32_t*>(at);
  if constexpr (N == 1) {
    w[0] = in ? __ldg(p) : 0u;
  } else if constexpr (N == 2) {
    const uint2 v = in ? __ldg(reinterpret_cast<const uint2*>(p)) : make_uint2(0, 0);
    w[0] = v.x; w[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint4 v = in ? ldg16(p + i) : make_uint4(0, 0, 0, 0);
      w[i] = v.x; w[i + 1] = v.y; w[i + 2] = v.z; w[i + 3] = v.w;
    }
  }
}

// bf16 number i of packed words, as float32.
template <int N> __device__ __forceinline__ float scale_at(const uint32_t (&w)[N], int i) {
  return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
}

constexpr uint32_t kEven = 0x000f000fu, kOdd = 0x00f000f0u;   // n 2^-24, n 2^-20 as f16

template <typename T, int D>
__global__ void __launch_bounds__(kAttendWarps * 32, D == 256 ? 1 : 2)
attend_kernel(const AttendParams<T> p) {
  constexpr int NG = D / kGroup;                     // groups of a row
  constexpr int QP = sizeof(T) == 4 ? 3 : 1;         // f16 parts of the query
  constexpr int VP = sizeof(T) == 4 ? 3 : 2;         // f16 parts of a weight
  constexpr int VC = VP == 3 ? 4 : 2;                // B columns of a group
  constexpr int GT = 8 / VC;                         // groups per set of 8 columns
  constexpr int NV = (NG + GT - 1) / GT;             // sets of columns
  constexpr int KW = D / 32, VW = D / 64;            // words per lane of a key / value row
  constexpr int MT = D / 16;                         // tiles of 16 output elements
  constexpr int E = Vec<T>::kElems;
  __shared__ float s_ml[kAttendWarps][2];
  __shared__ __align__(16) float s_out[kAttendWarps][D];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int wpp = p.warps_per_pair, sub = warp % wpp;
  // pairs in the order [B, Hkv, L, G]: neighbouring warps read neighbouring keys
  const int64_t pair = (int64_t)blockIdx.x * (kAttendWarps / wpp) + warp / wpp;
  const bool live = pair < p.pairs;
  const int64_t pr = live ? pair : p.pairs - 1;
  const int64_t rest = pr / p.G, bh = rest / p.span.L;
  const int64_t l = rest % p.span.L;
  const int hkv = (int)(bh % p.c.Hkv), b = (int)(bh / p.c.Hkv);
  const int h = hkv * p.G + (int)(pr % p.G);
  const int pos = live ? (int)p.span.position(b, l, p.c.S) : -1;   // < 2^24
  if (pos == -2 && sub == 0 && lane == 0 && p.err) atomicOr(p.err, kErrQueryRange);

  // The query as B columns 0 .. QP - 1: this lane's 8 elements of each group, as
  // the nibbles of a word pair up: (0, 4), (1, 5) / 16, (2, 6), (3, 7) / 16.
  uint32_t qb[NG][4];
  float qoff[NG];                                    // what the codes' + 8 adds
  float unit;                                        // of the scores
  {
    float f[NG][8];
    uint32_t top = 0;
    const T* q = static_cast<const T*>(p.q.data) + b * p.q.sb + h * p.q.sh + l * p.q.ss + t * 8;
#pragma unroll
    for (int c = 0; c < NG; ++c) {
#pragma unroll
      for (int i = 0; i < 8; i += E) Vec<T>::to_float(ldg16(q + c * kGroup + i), f[c] + i);
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max(top, int4::abs_bits(f[c][i]));
    }
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    float down;
    const float up = lift(min(top, 0x7f7fffffu), down);
    unit = down * p.scale_log2;
#pragma unroll
    for (int c = 0; c < NG; ++c) {
      float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float f16 = i & 1 ? up * 0.0625f : up;
        qb[c][i] = half_part<QP>(f[c][i] * f16, f[c][i + 4] * f16, g);
      }
      // 1 and 16 in f16: the sum of the group
      mma(s, 0x3c003c00u, 0x3c003c00u, 0x4c004c00u, 0x4c004c00u, qb[c][0], qb[c][1]);
      mma(s, 0x3c003c00u, 0x3c003c00u, 0x4c004c00u, 0x4c004c00u, qb[c][2], qb[c][3]);
      qoff[c] = (s[0] + s[1]) * 0x1p-21f;
    }
  }

  const RowWin rw = row_window(p.pat, pos < 0 ? 0 : pos);
  const float ht = head_weight(p.pat, h), omt = __fsub_rn(1.f, ht);
  const int64_t row0 = ((int64_t)b * p.c.Hkv + hkv) * p.c.S;
  const uint8_t* codes = p.c.codes + row0 * D;
  const __nv_bfloat16* scales = p.c.scales + row0 * (2 * NG);
  const int nchunks = pos < 0 ? 0 : (p.pat.w + 31) >> 5;

  // this lane's columns in the output products: column set nv holds group
  // nv * GT + g / VC, part g % VC; results in columns 2 t and 2 t + 1
  const int owner = VC == 2 ? t : t >> 1;
  float total[NV][2][2];
#pragma unroll
  for (int i = 0; i < NV * 4; ++i) (&total[0][0][0])[i] = 0.f;
  float m_run = -INFINITY, l_run = 0.f;

  for (int chunk = sub; chunk < nchunks; chunk += wpp) {
    const int slot = chunk * 32 + lane;
    int myrow = -1;
    if (slot < p.pat.w) {
      const int raw = raw_index(rw, slot, ht, omt);
      if (raw <= pos && raw >= 0) myrow = raw;       // causal
    }
    if (__ballot_sync(0xffffffffu, myrow >= 0) == 0) continue;
    // ---- all loads of the 32 slots ----
    uint32_t kw[2][2][KW], ks[2][2][NG / 2], vw[2][4][VW];
    float vs[2][4][NV];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = __shfl_sync(0xffffffffu, myrow, i * 16 + r * 8 + g);
        load_words<KW>(codes + (int64_t)row * D + t * (KW * 4), row >= 0, kw[i][r]);
        load_words<NG / 2>(scales + (int64_t)row * (2 * NG), row >= 0, ks[i][r]);
      }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int row = __shfl_sync(0xffffffffu, myrow, i * 16 + 2 * t + (k & 1) + (k >> 1) * 8);
        load_words<VW>(codes + (int64_t)row * D + D / 2 + g * (VW * 4), row >= 0, vw[i][k]);
#pragma unroll
        for (int nv = 0; nv < NV; ++nv) {
          const int gi = nv * GT + g / VC;
          vs[i][k][nv] = row >= 0 && gi < NG
                             ? __bfloat162float(scales[(int64_t)row * (2 * NG) + NG + gi]) : 0.f;
        }
      }
    // ---- scores ----
    float sc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      sc[i][0] = sc[i][1] = 0.f;
#pragma unroll
      for (int c = 0; c < NG; ++c) {
        float a[4] = {0.f, 0.f, 0.f, 0.f};
        const uint32_t x = kw[i][0][c], y = kw[i][1][c], x8 = x >> 8, y8 = y >> 8;
        mma(a, x & kEven, y & kEven, x & kOdd, y & kOdd, qb[c][0], qb[c][1]);
        mma(a, x8 & kEven, y8 & kEven, x8 & kOdd, y8 & kOdd, qb[c][2], qb[c][3]);
        sc[i][0] = fmaf(scale_at(ks[i][0], c), a[0] + a[1] - qoff[c], sc[i][0]);
        sc[i][1] = fmaf(scale_at(ks[i][1], c), a[2] + a[3] - qoff[c], sc[i][1]);
      }
      if constexpr (QP == 3) {                        // the third part is with lane t = 1
        sc[i][0] += __shfl_xor_sync(0xffffffffu, sc[i][0], 1);
        sc[i][1] += __shfl_xor_sync(0xffffffffu, sc[i][1], 1);
      }
    }
    // lanes t = 0 hold slots g and g + 8 of each 16: one slot per lane
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float v = __shfl_sync(0xffffffffu, sc[i][r], (lane & 7) * 4);
        if ((lane >> 3) == i * 2 + r) s = v;
      }
    s = myrow >= 0 ? s * 0x1p24f * unit : -INFINITY;
    const float mn = fmaxf(m_run, warp_max(s));
    const float ref = mn == -INFINITY ? 0.f : mn;
    const float corr = exp2f(m_run - ref);            // 0 on the first chunk
    const float e = exp2f(s - ref);
    l_run = l_run * corr + warp_sum(e);
    m_run = mn;
    // ---- weighted values ----
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float w = __shfl_sync(0xffffffffu, e, i * 16 + 2 * t + (k & 1) + (k >> 1) * 8);
#pragma unroll
        for (int nv = 0; nv < NV; ++nv) {
          vs[i][k][nv] *= w;
          top = fmaxf(top, vs[i][k][nv]);             // passes over NaN
        }
      }
    float down;
    const float up = lift(__reduce_max_sync(0xffffffffu, min(__float_as_uint(top), 0x7f7fffffu)), down);
    float acc[MT][4], ones[NV][4];
#pragma unroll
    for (int i = 0; i < MT * 4; ++i) (&acc[0][0])[i] = 0.f;
#pragma unroll
    for (int i = 0; i < NV * 4; ++i) (&ones[0][0])[i] = 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t vb[NV][2];
#pragma unroll
      for (int nv = 0; nv < NV; ++nv) {
        vb[nv][0] = half_part<VP>(vs[i][0][nv] * up, vs[i][1][nv] * up, g % VC);
        vb[nv][1] = half_part<VP>(vs[i][2][nv] * up, vs[i][3][nv] * up, g % VC);
        mma(ones[nv], 0x00010001u, 0x00010001u, 0x00010001u, 0x00010001u, vb[nv][0], vb[nv][1]);
      }
#pragma unroll
      for (int c = 0; c < VW; ++c)
#pragma unroll
        for (int half = 0; half < 2; ++half) {        // nibbles 0 .. 3, 4 .. 7: 32 elements, one group
          const uint32_t sel = half ? 0x7632u : 0x5410u;
          const uint32_t x = __byte_perm(vw[i][0][c], vw[i][1][c], sel), x8 = x >> 8;
          const uint32_t y = __byte_perm(vw[i][2][c], vw[i][3][c], sel), y8 = y >> 8;
          const int gr = 2 * c + half, nv = gr / GT;
          mma(acc[2 * gr], x & kEven, x & kOdd, y & kEven, y & kOdd, vb[nv][0], vb[nv][1]);
          mma(acc[2 * gr + 1], x8 & kEven, x8 & kOdd, y8 & kEven, y8 & kOdd, vb[nv][0], vb[nv][1]);
        }
    }
    // the columns of this lane belong to one group of each set
#pragma unroll
    for (int nv = 0; nv < NV; ++nv) {
      const float off = 8.f * (ones[nv][0] + ones[nv][1]);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float lo = 0.f, hi = 0.f;
#pragma unroll
        for (int o = 0; o < GT; ++o) {
          const int gr = nv * GT + o;
          if (gr < NG && owner == o) {
            lo = acc[2 * (gr < NG ? gr : 0) + j][0] + acc[2 * (gr < NG ? gr : 0) + j][1];
            hi = acc[2 * (gr < NG ? gr : 0) + j][2] + acc[2 * (gr < NG ? gr : 0) + j][3];
          }
        }
        total[nv][j][0] = fmaf(lo - off, down, total[nv][j][0] * corr);
        total[nv][j][1] = fmaf(fmaf(hi, 0.0625f, -off), down, total[nv][j][1] * corr);
      }
    }
  }

  // ---- the warps of a pair ----
#pragma unroll
  for (int nv = 0; nv < NV; ++nv)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float v = total[nv][j][r] * 0x1p24f;
        if constexpr (VC == 4) v += __shfl_xor_sync(0xffffffffu, v, 1);
        const int gr = nv * GT + owner;
        if (gr < NG && (VC == 2 || (t & 1) == 0))
          s_out[warp][gr * kGroup + j * 16 + r * 8 + g] = v;
      }
  if (lane == 0) {
    s_ml[warp][0] = m_run;
    s_ml[warp][1] = l_run;
  }
  if (wpp > 1) __syncthreads(); else __syncwarp();
  if (sub != 0 || !live) return;
  float mx = -INFINITY;
  for (int i = 0; i < wpp; ++i) mx = fmaxf(mx, s_ml[warp + i][0]);
  const float ref = mx == -INFINITY ? 0.f : mx;
  float sum = 0.f;
  constexpr int PL = D / 32;                          // elements per lane
  float out[PL];
#pragma unroll
  for (int i = 0; i < PL; ++i) out[i] = 0.f;
  for (int i = 0; i < wpp; ++i) {
    const float f = exp2f(s_ml[warp + i][0] - ref);
    sum = fmaf(s_ml[warp + i][1], f, sum);
#pragma unroll
    for (int e = 0; e < PL; ++e) out[e] = fmaf(s_out[warp + i][lane * PL + e], f, out[e]);
  }
  const float inv = sum != 0.f ? 1.f / sum : 0.f;
  T* o = static_cast<T*>(const_cast<void*>(p.o.data)) + b * p.o.sb + h * p.o.sh + l * p.o.ss + lane * PL;
  struct alignas(PL * sizeof(T) < 16 ? PL * sizeof(T) : 16) Pack { T v[PL]; } pack;
#pragma unroll
  for (int e = 0; e < PL; ++e) pack.v[e] = from_f32<T>(out[e] * inv);
  *reinterpret_cast<Pack*>(o) = pack;
  if (lane == 0) p.lse[((int64_t)b * p.Hq + h) * p.span.L + l] = ref + log2f(sum);
}

}  // namespace cache4
}  // namespace esa
