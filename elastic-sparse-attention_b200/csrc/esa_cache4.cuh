// Keys and values cached in 4 bits (esa_int4.cuh, groups of 32 along the head
// dimension) and the elastic attention that reads them.
//
// A cached row of one K/V head is D / 2 bytes of key codes, D / 2 bytes of value
// codes (one 128-byte line for D = 128) and 2 x D / 32 bf16 scales.  The codes
// lie in the order in which the matrix instructions take them:
//   key:   word t * (D / 32) + c of a row (t < 4, c < D / 32) holds the elements
//          (c / 2) * 64 + (i & 1) * 32 + t * 8 + (c & 1) * 4 + i / 2, nibble i: the low
//          nibbles of two words are one group, the high ones the next; the nibbles
//          of keys are two's complement (the code, not code + 8)
//   value: word g * (D / 64) + c (g < 8, c < D / 64) holds the elements
//          c * 64 + i * 8 + g, nibble i
// and the 32-byte sectors of a row are turned by its number (turn_of), so that
// lanes which read the same part of different rows mostly meet different banks.
//
// Attention: every (query row, head) pair has w keys of its own, so nothing is
// shared between pairs and the work is decoding 2 w D codes.  The products run
// on mma.sync m16n8k32 of 8-bit integers (exact, the same rate as f16 with twice
// the elements) with the stored codes (n = code + 8, one AND per four) as A and
// the query, or the softmax weights, as fixed-point numbers in the columns of B
// that one vector leaves free otherwise, a column per digit of 8 bits:
//   scores: A = 16 keys x 32 elements (one group), B column = digit of the query,
//           four digits (30 bits below the query's largest element); the sum of a
//           group times its scale in float32
//   output: A = 16 elements x 32 keys, B column = (group, digit) of the weight
//           times that group's scale, two digits (16 bits below the largest of
//           the 32 keys in that group) for 16-bit types and four for float32; an
//           output element reads the columns of its group
// Keys are signed bytes, 16 times the code; what the stored + 8 of the values adds
// is taken out exactly by one product with a matrix of eights.
// (f16 products with the nibbles as denormals need as little decoding, but lose
// 9 bits when the tensor core aligns them: the output was 2^-11 off.)
//
// Measured: 4096 rows x 32 heads of 128, w = 64, at the end of 131072 positions:
// 212 us (esa_forward on a 16-bit cache of that shape: 444; 206 with one grid of weights
// for all groups of a head, on which a group 4096 times smaller than the largest was
// a tenth off); some 1290 instructions a pair fill 73 % of the issue slots, the integer
// pipe 67 %.  8 single rows: 3.6 us.
// Rows in: 79 us, out: 62 us for 3 x 20011 x 8 rows of 128 fp16 (profiled; together 138
// without), bound by instructions: 78 and 74 % of the issue slots, DRAM at 25 and 50 %.
//
// A warp takes 32 slots of a pair at a time, all their loads in flight, with an
// online softmax in float32; with few pairs a pair's slots are split over the
// warps of a CTA and joined in shared memory.
#pragma once
#include "esa_int4.cuh"
#include "esa_pack8.cuh"

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
};

// What the byte offsets within a row of 128-byte lines are combined with by XOR.
template <int D> __device__ __forceinline__ uint32_t turn_of(uint32_t row) {
  return D == 64 ? (row & 2u) << 4 : (row & 3u) << 5;
}

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
// Rows into the cache and out of it.  A thread owns 8 elements of a head row of k and
// of v; D / 8 neighbouring threads a row; rows in the order [L, H], as a projection
// leaves them, two per thread so that twice the loads are on their way.
// ---------------------------------------------------------------------------
struct Heads { const void* data; int64_t sb, sh, ss; };

constexpr int kRowThreads = 256, kRowsPerThread = 2;

template <typename T> struct RowParams {
  Cache c;
  Span span;
  Heads k, v;
  unsigned rows;              // L * Hkv, of one sequence (blockIdx.y)
  int* err;
};

template <int D> struct Unit {          // which 8 elements a thread owns
  static constexpr int kPer = D / 8, kRows = kRowThreads / kPer;       // rows of a CTA at a time
  int l, pos, h;
  bool in, go;                          // a row of the call; one that lies in the cache
  // Rows [lo, hi) of the sequence have positions begin + l in the cache.
  __device__ __forceinline__ void set(unsigned r, unsigned rows, unsigned heads, int begin, int lo,
                                      int hi) {
    in = r < rows;
    const unsigned q = in ? r : rows - 1;
    l = (int)(q / heads);
    h = (int)(q - (unsigned)l * heads);
    pos = begin + l;
    go = in && l >= lo && l < hi;
  }
};

// The units of a thread, and the part of the rows that it owns.
template <int D> struct Units {
  Unit<D> u[kRowsPerThread];
  int part;
  template <typename T>
  __device__ __forceinline__ explicit Units(const RowParams<T>& p) {
    part = threadIdx.x % Unit<D>::kPer;
    const int64_t begin = p.span.begin(blockIdx.y), count = p.span.count(blockIdx.y);
    // begin is clamped to a place from which no row lies in the cache, so that 32 bits hold
    // it: the cache's end, or as many positions before its begin as the call has rows
    const int first = (int)(begin < -p.span.L ? -p.span.L : begin > p.c.S ? p.c.S : begin);
    const int n = (int)count, lo = first < 0 ? min(-first, n) : 0;
    const int hi = max(min(n, (int)p.c.S - first), lo);
    if ((lo > 0 || hi < n) && threadIdx.x == 0 && blockIdx.x == 0 && p.err) atomicOr(p.err, kErrKvRange);
#pragma unroll
    for (int i = 0; i < kRowsPerThread; ++i)
      u[i].set((blockIdx.x * kRowsPerThread + i) * Unit<D>::kRows + threadIdx.x / Unit<D>::kPer, p.rows,
               (unsigned)p.c.Hkv, first, lo, hi);
  }
  // The words of keys hold 4 elements of this thread and 4 of the thread with the
  // next group: two words, shared by two threads.
  __device__ __forceinline__ int key_word(int i) const {
    return ((part & 3) * (D / 32) + (part >> 3) * 2 + (part >> 2 & 1)) ^ turn(i);
  }
  __device__ __forceinline__ int value_word(int i) const {
    return (D / 8 + (part & 7) * (D / 64) + (part >> 3)) ^ turn(i);
  }
  __device__ __forceinline__ int turn(int i) const { return (int)turn_of<D>((uint32_t)u[i].pos) / 4; }
  __device__ __forceinline__ int64_t row(const Cache& c, int i) const {
    return (int64_t)(blockIdx.y * (unsigned)c.Hkv + (unsigned)u[i].h) * c.S + u[i].pos;
  }
  template <typename T> __device__ __forceinline__ T* address(const Heads& x, int i) const {
    return static_cast<T*>(const_cast<void*>(x.data)) + blockIdx.y * x.sb + u[i].h * x.sh +
           u[i].l * x.ss + part * 8;
  }
};

// Largest magnitudes (float bits, NaN above infinity above finite) of the groups of
// two times 8 elements, a group being 4 neighbouring lanes.  16-bit types compare two
// elements per instruction and carry both groups through one chain of shuffles.
template <typename T>
__device__ __forceinline__ void group_max(const uint4 (&x)[2][sizeof(T) / 2], uint32_t (&top)[2]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      uint32_t m = 0;
#pragma unroll
      for (int n = 0; n < 2; ++n)
        m = max(max(m, max(x[j][n].x & 0x7fffffffu, x[j][n].y & 0x7fffffffu)),
                max(x[j][n].z & 0x7fffffffu, x[j][n].w & 0x7fffffffu));
      m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
      top[j] = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
    }
  } else {
    using M = pack8::Max2<T>;
    uint32_t m[2];
#pragma unroll
    for (int j = 0; j < 2; ++j)
      m[j] = M::abs_max(M::abs_max(x[j][0].x, x[j][0].y), M::abs_max(x[j][0].z, x[j][0].w));
    uint32_t r = M::abs_max(__byte_perm(m[0], m[1], 0x5410), __byte_perm(m[0], m[1], 0x7632));
    r = M::abs_max(r, __shfl_xor_sync(0xffffffffu, r, 1));
    r = M::abs_max(r, __shfl_xor_sync(0xffffffffu, r, 2));
    top[0] = pack8::magnitude_bits<T>(r);
    top[1] = pack8::magnitude_bits<T>(r >> 16);
  }
}

// Codes (one nibble each) of 8 elements, and their group's scale.
template <typename T>
__device__ __forceinline__ uint32_t encode8(const uint4 (&v)[sizeof(T) / 2], uint32_t top, float& s) {
  float f[8], inv;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) Vec<T>::to_float(v[i], f + i * Vec<T>::kElems);
  s = int4::group_scale(top, inv);
  return int4::codes_of<T>(f, s, inv);
}

// Two threads, four lanes apart, with the nibbles of their 8 elements <-> the first
// (second) of the two key words that hold them.
__device__ __forceinline__ uint32_t mix_keys(uint32_t w, int part) {
  const uint32_t o = __shfl_xor_sync(0xffffffffu, w, 4);
  const uint32_t a = part & 4 ? o : w, b = part & 4 ? w : o;      // the lower group, the higher
  // the first word takes nibbles 0 .. 3 of both, the second 4 .. 7
  const uint32_t x = part & 4 ? a >> 16 : a & 0xffffu, y = part & 4 ? b >> 16 : b & 0xffffu;
  auto spread = [](uint32_t v) {                                  // nibbles to bytes
    v = (v | v << 8) & 0x00ff00ffu;
    return (v | v << 4) & 0x0f0f0f0fu;
  };
  return spread(x) | spread(y) << 4;
}
__device__ __forceinline__ uint32_t unmix_keys(uint32_t w, int part) {
  const uint32_t o = __shfl_xor_sync(0xffffffffu, w, 4);
  const uint32_t a = part & 4 ? o : w, b = part & 4 ? w : o;      // the first word, the second
  auto gather = [](uint32_t v) {                                  // low nibbles of bytes together
    v &= 0x0f0f0f0fu;
    v = (v | v >> 4) & 0x00ff00ffu;
    return (v | v >> 8) & 0xffffu;
  };
  const int s = part & 4 ? 4 : 0;
  return gather(a >> s) | gather(b >> s) << 16;
}

template <typename T, int D>
__global__ void __launch_bounds__(kRowThreads)
write_kernel(const RowParams<T> p) {
  constexpr int N = sizeof(T) / 2;                     // 16-byte vectors of 8 elements
  const Units<D> u(p);
  uint4 x[kRowsPerThread][2][N];
#pragma unroll
  for (int i = 0; i < kRowsPerThread; ++i) {
    const T* k = u.template address<T>(p.k, i);
    const T* v = u.template address<T>(p.v, i);
#pragma unroll
    for (int n = 0; n < N; ++n) {
      x[i][0][n] = x[i][1][n] = make_uint4(0, 0, 0, 0);
      if (u.u[i].go) {
        x[i][0][n] = ldg16_stream(k + n * Vec<T>::kElems);
        x[i][1][n] = ldg16_stream(v + n * Vec<T>::kElems);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kRowsPerThread; ++i) {
    float sk, sv;
    uint32_t top[2];
    group_max<T>(x[i], top);
    const uint32_t kw = mix_keys(encode8<T>(x[i][0], top[0], sk), u.part) ^ 0x88888888u;
    const uint32_t vw = transpose8(encode8<T>(x[i][1], top[1], sv), u.part & 7);
    if (!u.u[i].go) continue;
    const int64_t row = u.row(p.c, i);
    uint32_t* codes = reinterpret_cast<uint32_t*>(p.c.codes + row * D);
    codes[u.key_word(i)] = kw;
    codes[u.value_word(i)] = vw;
    if ((u.part & 3) == 0) {
      __nv_bfloat16* s = p.c.scales + row * (2 * D / kGroup) + (u.part >> 2);
      s[0] = __float2bfloat16_rn(sk);
      s[D / kGroup] = __float2bfloat16_rn(sv);
    }
  }
}

// Rows outside the cache come out as zeros.
template <typename T, int D>
__global__ void __launch_bounds__(kRowThreads)
read_kernel(const RowParams<T> p) {
  constexpr int N = sizeof(T) / 2;
  const Units<D> u(p);
  uint32_t w[kRowsPerThread][2];
  float s[kRowsPerThread][2];
#pragma unroll
  for (int i = 0; i < kRowsPerThread; ++i) {
    w[i][0] = 0u;
    w[i][1] = 0x88888888u;
    s[i][0] = s[i][1] = 0.f;
    if (u.u[i].go) {
      const int64_t row = u.row(p.c, i);
      const uint32_t* codes = reinterpret_cast<const uint32_t*>(p.c.codes + row * D);
      w[i][0] = __ldg(codes + u.key_word(i));
      w[i][1] = __ldg(codes + u.value_word(i));
      const __nv_bfloat16* f = p.c.scales + row * (2 * D / kGroup) + (u.part >> 2);
      s[i][0] = __bfloat162float(f[0]);
      s[i][1] = __bfloat162float(f[D / kGroup]);
    }
  }
#pragma unroll
  for (int i = 0; i < kRowsPerThread; ++i) {
    const uint32_t kv[2] = {unmix_keys(w[i][0], u.part) ^ 0x88888888u, transpose8(w[i][1], u.part & 7)};
    if (!u.u[i].in) continue;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      T* to = u.template address<T>(j ? p.v : p.k, i);
      uint32_t out[4 * N];
      int4::decode8<T>(kv[j], s[i][j], out);
#pragma unroll
      for (int n = 0; n < N; ++n)
        stg16(to + n * Vec<T>::kElems, make_uint4(out[4 * n], out[4 * n + 1], out[4 * n + 2], out[4 * n + 3]));
    }
  }
}

// ---------------------------------------------------------------------------
// Attention.
// ---------------------------------------------------------------------------
// d = A B, m16n8k32 of 8-bit integers, both signed or both unsigned.  The
// instructions that all lanes of a warp execute together are volatile: without it
// the compiler may move one under a condition that only uses its result on some
// lanes, where it waits for the others for good.
template <bool SIGNED>
__device__ __forceinline__ void mma(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                    const uint32_t (&b)[2]) {
#define ESA_MMA(T)                                                                          \
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32." T "." T ".s32 {%0,%1,%2,%3}, "      \
               "{%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"                                 \
               : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])                             \
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b[0]), "r"(b[1]), "r"(0))
  if constexpr (SIGNED) ESA_MMA("s8");
  else ESA_MMA("u8");
#undef ESA_MMA
}

// Largest of the warp's values (a NaN is above all): their bits in the order of
// signed integers.
__device__ __forceinline__ float max_of_warp(float x) {
  const int b = __float_as_int(x);
  const int m = __reduce_max_sync(0xffffffffu, b ^ ((b >> 31) & 0x7fffffff));
  return __int_as_float(m ^ ((m >> 31) & 0x7fffffff));
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 2^e with x 2^e in [2^TOP, 2^(TOP + 1)) for the float bits of x >= 0 (2^126 where x
// is 0 or too small for that), and its inverse.  (Of an infinity or a NaN: some finite
// power.)  SHRINK: the power is 1 - 2^-16 times that, 256 units of its last place less.
template <int TOP, bool SHRINK = false>
__device__ __forceinline__ float lift(uint32_t bits, float& inverse) {
  constexpr uint32_t kLess = SHRINK ? 256u : 0u;
  const uint32_t up = min((253u << 23) - kLess, ((TOP + 254u) << 23) - kLess - (bits & 0x7f800000u));
  inverse = __uint_as_float((254u << 23) - kLess - up);
  return __uint_as_float(up);
}

// Byte j of four words, in x[j].
__device__ __forceinline__ void transpose_bytes(const uint32_t (&w)[4], uint32_t (&x)[4]) {
  const uint32_t a = __byte_perm(w[0], w[1], 0x5140), b = __byte_perm(w[2], w[3], 0x5140);
  const uint32_t c = __byte_perm(w[0], w[1], 0x7362), d = __byte_perm(w[2], w[3], 0x7362);
  x[0] = __byte_perm(a, b, 0x5410);
  x[1] = __byte_perm(a, b, 0x7632);
  x[2] = __byte_perm(c, d, 0x5410);
  x[3] = __byte_perm(c, d, 0x7632);
}

template <typename T> struct AttendParams {
  Cache c;
  Span span;
  Heads q, o;
  int Hq, G;                  // query heads, query heads per K/V head
  unsigned rows;              // G * L: pairs of one K/V head
  int warps_per_pair;         // 1, 2 or 4
  int pairs_per_warp;         // one after the other; 1 where warps share a pair
  Pattern pat;
  float scale_log2;
  float* lse;                 // [B, Hq, L]
  int* err;
};

constexpr int kAttendWarps = 4;

// row_window with inv_w = f32(1 / w): the quotient of two integers is rounded
// correctly by one step from q = n inv_w with the exact remainder n - q w (Markstein,
// IBM J. Res. Dev. 34, 1990), without the branches of a general division.
__device__ __forceinline__ RowWin row_window_inv(const Pattern& P, int pos, float inv_w) {
  const int end = pos > P.w - 1 ? pos : P.w - 1;
  const float E = __int2float_rn(end + 1);
  const float pd = __fadd_rn(P.c, __fmul_rn(E, P.a));
  const float s = fmaxf(rintf(__fsub_rn(E, pd)), 0.f);
  RowWin r;
  r.st = __float2int_rz(s);
  const float n = __int2float_rn(end + 1 - r.st), w = __int2float_rn(P.w);
  const float q = __fmul_rn(n, inv_w);
  r.sp = fmaf(fmaf(-w, q, n), inv_w, q);
  return r;
}

template <int N> __device__ __forceinline__ void load_words(const void* at, uint32_t (&w)[N]) {
  const uint32_t* p = static_cast<const uint32_t*>(at);
  if constexpr (N == 1) {
    w[0] = __ldg(p);
  } else if constexpr (N == 2) {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
    w[0] = v.x; w[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint4 v = ldg16(p + i);
      w[i] = v.x; w[i + 1] = v.y; w[i + 2] = v.z; w[i + 3] = v.w;
    }
  }
}

// bf16 number i of packed words, as float32.
template <int N> __device__ __forceinline__ float scale_at(const uint32_t (&w)[N], int i) {
  return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
}

// Nibbles as 8-bit numbers: the low ones n, the high ones 16 n, and what the + 8 of
// a value's code is then.
constexpr uint32_t kLow = 0x0f0f0f0fu, kHigh = 0xf0f0f0f0u;
constexpr uint32_t kEight = 0x08080808u, kEightHigh = 0x80808080u;     // 8, 128
// 1 / (1 - 2^-16), which two digits' weights are short of: taken once per output.
constexpr float kGrow = 1.00001525902189f;

// SPLIT: the warps of a CTA share pairs, one pair at a time; else each warp has
// pairs of its own, one after the other.
template <typename T, int D, bool SPLIT>
__global__ void __launch_bounds__(kAttendWarps * 32, D == 256 ? 2 : 5)
attend_kernel(const AttendParams<T> p) {
  constexpr int NG = D / kGroup;                     // groups of a row
  constexpr int VC = sizeof(T) == 4 ? 4 : 2;         // digits (B columns) of a weight
  constexpr int GT = 8 / VC;                         // groups per set of 8 columns
  constexpr int NV = (NG + GT - 1) / GT;             // sets of columns
  constexpr int KW = D / 32, VW = D / 64;            // words per lane of a key / value row
  constexpr int MT = D / 16;                         // tiles of 16 output elements
  constexpr int E = Vec<T>::kElems;
  constexpr int QS = NG * 8 + 8;                     // words of a digit's plane, offset by 8 banks
  __shared__ float s_ml[kAttendWarps][2];
  // query, then weights [group][digit][32 keys] in bytes, then output
  constexpr int BUF = 4 * QS > D ? 4 * QS : D;
  static_assert(NG * VC * 32 <= BUF * 4, "the digits of the weights fit the buffer");
  __shared__ __align__(16) uint32_t s_buf[kAttendWarps][BUF];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int wpp = SPLIT ? p.warps_per_pair : 1, sub = SPLIT ? warp & (wpp - 1) : 0;
  // grid = (pairs of a K/V head, B * Hkv); pairs in the order [G, L]: neighbouring
  // rows of a head attend to the same or neighbouring keys
  const unsigned L = (unsigned)p.span.L;
  const unsigned step = SPLIT ? (unsigned)(kAttendWarps / wpp) : kAttendWarps;   // pairs a CTA has at a time
  unsigned pair = blockIdx.x * step * (unsigned)p.pairs_per_warp + (unsigned)(SPLIT ? warp / wpp : warp);
  const int b = (int)(blockIdx.y / (unsigned)p.c.Hkv);
  int h = (int)(blockIdx.y % (unsigned)p.c.Hkv) * p.G + (int)(pair / L);
  unsigned l = pair % L;
  const int64_t begin = p.span.begin(b), count = p.span.count(b);
  const int64_t row0 = (int64_t)blockIdx.y * p.c.S;
  // rows of this K/V head lie within 2^32 bytes: max_len <= 2^24, D <= 256
  const uint8_t* codes = p.c.codes + row0 * D;
  const uint8_t* scales = reinterpret_cast<const uint8_t*>(p.c.scales + row0 * (2 * NG));
  const T* q = static_cast<const T*>(p.q.data) + b * p.q.sb;
  constexpr int SETS = (NG * 8 + 31) / 32;           // 4 elements of the query per lane and set
  using QV = typename std::conditional<E == 4, uint4, uint2>::type;
  QV qv[SETS];
  auto load_query = [&](bool in) {
#pragma unroll
    for (int i = 0; i < SETS; ++i) {
      const int set = i * 32 + lane;
      qv[i] = QV{};
      if (in && (NG * 8 % 32 == 0 || set < NG * 8))
        // o may be q: a pair's query is read before its output is written, and by an ordinary load
        qv[i] = *reinterpret_cast<const QV*>(q + h * p.q.sh + (int64_t)l * p.q.ss + set * 4);
    }
  };
  load_query(pair < p.rows);
  float ht = head_weight(p.pat, h), omt = __fsub_rn(1.f, ht);
  const float inv_w = __frcp_rn((float)p.pat.w);

  for (int it = 0; it < p.pairs_per_warp; ++it) {
  const bool live = pair < p.rows;
  if (!SPLIT && !live) break;
  const int my_h = h;
  const unsigned my_l = l;
  const float my_ht = ht, my_omt = omt;
  // < 2^24; padding and positions outside the cache have no slots
  const bool inside = begin >= 0 && begin < p.c.S - (int64_t)l;
  const int pos = live && inside && (int64_t)l < count ? (int)(begin + l) : -1;
  if (live && !inside && (int64_t)l < count && sub == 0 && lane == 0 && p.err)
    atomicOr(p.err, kErrQueryRange);

  // The query in fixed point, as columns of balanced digits -128 .. 127.  Four
  // neighbouring elements of one lane make a B word; shared memory brings the words
  // of digit g to lanes 4 g + t.
  uint32_t qb[NG][2];
  float unit;                                        // of the scores
  {
    float f[SETS][4];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < SETS; ++i) {
      if constexpr (E == 4) {
        Vec<T>::to_float(qv[i], f[i]);
      } else {
        float w[8];
        Vec<T>::to_float(make_uint4(qv[i].x, qv[i].y, 0u, 0u), w);
#pragma unroll
        for (int k = 0; k < 4; ++k) f[i][k] = w[k];
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) top = max(top, int4::abs_bits(f[i][k]));
    }
    // the next pair's query is on its way while this one is worked on
    pair += step;
    l += step;
    if (l >= L) {
      do {
        l -= L;
        ++h;
      } while (l >= L);
      ht = head_weight(p.pat, h);
      omt = __fsub_rn(1.f, ht);
    }
    if (it + 1 < p.pairs_per_warp) load_query(pair < p.rows);
    top = __reduce_max_sync(0xffffffffu, top);
    float down;
    const float up = lift<29>(min(top, 0x7f7fffffu), down);
    // an infinity or a NaN in the query: no score is a number
    unit = top >= 0x7f800000u ? __uint_as_float(0x7fffffffu) : down * 0.0625f * p.scale_log2;
#pragma unroll
    for (int i = 0; i < SETS; ++i) {
      // digits are the bytes of x + 0x80808080, less 0x80 each
      uint32_t d[4], x[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) d[k] = (uint32_t)__float2int_rn(f[i][k] * up) + 0x80808080u;
      transpose_bytes(d, x);
      if (NG * 8 % 32 == 0 || i * 32 + lane < NG * 8)
#pragma unroll
        for (int k = 0; k < 4; ++k) s_buf[warp][k * QS + i * 32 + lane] = x[k] ^ 0x80808080u;
    }
    __syncwarp();
#pragma unroll
    for (int c = 0; c < NG; ++c) {
      uint2 v = make_uint2(0, 0);                    // no digits in columns 4 .. 7
      if (g < 4) v = *reinterpret_cast<const uint2*>(&s_buf[warp][g * QS + c * 8 + t * 2]);
      qb[c][0] = v.x;
      qb[c][1] = v.y;
    }
    __syncwarp();                                    // the buffer is used again
  }
  const float digit_unit = t == 1 ? 65536.f : 1.f;   // t = 0 has digits 0 and 1, t = 1 the others

  const RowWin rw = row_window_inv(p.pat, pos < 0 ? 0 : pos, inv_w);
  const int nchunks = pos < 0 ? 0 : (p.pat.w + 31) >> 5;

  // this lane's columns in the output products: column set nv holds group
  // nv * GT + g / VC, digit g % VC; results in columns 2 t and 2 t + 1
  const int owner = VC == 2 ? t : t >> 1;
  float total[NV][2][2];
  uint32_t nans = 0;                                 // groups of values with a NaN
#pragma unroll
  for (int i = 0; i < NV * 4; ++i) (&total[0][0][0])[i] = 0.f;
  float m_run = -INFINITY, l_lane = 0.f;

  for (int chunk = sub; chunk < nchunks; chunk += wpp) {
    // lane (g, t) looks after slot t * 8 + g
    const int slot = chunk * 32 + t * 8 + g;
    const int raw = raw_index(rw, slot, my_ht, my_omt);
    const bool valid = slot < p.pat.w && raw <= pos && raw >= 0;   // causal
    const uint32_t any = __ballot_sync(0xffffffffu, valid);
    if (any == 0) continue;
    // masked slots read the row of one that is not: what they hold is in use anyway
    const int safe = __shfl_sync(0xffffffffu, raw, __ffs(any) - 1);
    const int myrow = valid ? raw : safe;
    // ---- all loads of the 32 slots ----
    uint32_t kw[4][KW], sw[NG], vw[8][VW];           // sw: the own key's scales, its value's scales
    const uint32_t at = (uint32_t)myrow * (uint32_t)D | turn_of<D>((uint32_t)myrow);
#pragma unroll
    for (int k = 0; k < 4; ++k) {                    // keys k * 8 + g
      const uint32_t row = __shfl_sync(0xffffffffu, at, (lane & 28) + k);
      load_words<KW>(codes + (row ^ (uint32_t)(t * (KW * 4))), kw[k]);
    }
    load_words<NG>(scales + (uint32_t)myrow * (uint32_t)(NG * 4), sw);
#pragma unroll
    for (int k = 0; k < 8; ++k) {                    // keys t * 8 + k
      const uint32_t row = __shfl_sync(0xffffffffu, at, k * 4 + t);
      load_words<VW>(codes + (row ^ (uint32_t)(D / 2 + g * (VW * 4))), vw[k]);
    }
    // ---- scores ----
    float sc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < NG; c += 2) {
      uint32_t f[4];                                 // scales of groups c and c + 1 of keys k * 8 + g
#pragma unroll
      for (int k = 0; k < 4; ++k) f[k] = __shfl_sync(0xffffffffu, sw[c / 2], (lane & 28) + k);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          // 16 times the codes as signed bytes
          int a[4];
          const int up = u ? 1 : 16;
          mma<true>(a, kw[2 * i][c] * up & kHigh, kw[2 * i + 1][c] * up & kHigh,
                    kw[2 * i][c + 1] * up & kHigh, kw[2 * i + 1][c + 1] * up & kHigh, qb[c + u]);
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const uint32_t w = f[2 * i + r];
            sc[2 * i + r] = fmaf(__uint_as_float(u ? w & 0xffff0000u : w << 16),
                                 (float)(a[2 * r] + a[2 * r + 1] * 256), sc[2 * i + r]);
          }
        }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) sc[k] *= digit_unit;
    transpose_reduce<4>(sc, lane);                   // lane (g, t): slot t * 8 + g
    const float s = valid ? sc[0] * unit : -INFINITY;
    const float mn = fmaxf(m_run, max_of_warp(s));
    const float ref = mn == -INFINITY ? 0.f : mn;
    const float corr = ex2(m_run - ref);              // 0 on the first chunk
    const float e = ex2(s - ref);
    l_lane = fmaf(l_lane, corr, e);
    m_run = mn;
    // ---- weight times the scales of the own key's value, in fixed point: each group
    // on a grid of its own, since its outputs are no other group's ----
    float down[NV];                                  // of the groups this lane's columns hold
    uint32_t top[NG];
    unsigned char* digits = reinterpret_cast<unsigned char*>(s_buf[warp]);
#pragma unroll
    for (int c = 0; c < NG; ++c) {
      const uint32_t w = sw[(NG + c) / 2];
      // a masked slot's scale is one that is in use, so 0 times it is 0 or a NaN that
      // the key in use brings anyway
      const float vs = e * __uint_as_float(c & 1 ? w & 0xffff0000u : w << 16);
      top[c] = __reduce_max_sync(0xffffffffu, __float_as_uint(vs));   // none is negative
      // two digits: at most 65535 after the rounding
      float inverse;
      const float up = lift<VC == 4 ? 31 : 15, VC == 2>(top[c], inverse);
      if (c % GT == 0 || owner == c % GT) down[c / GT] = inverse;
      uint32_t d;
      // the product plus 2^23 has the rounded product as its low bits
      if constexpr (VC == 2) d = __float_as_uint(fmaf(vs, up, 8388608.f));
      else d = __float2uint_rn(vs * up);
#pragma unroll
      for (int i = 0; i < VC; ++i) digits[(c * VC + i) * 32 + t * 8 + g] = (unsigned char)(d >> (8 * i));
    }
    uint32_t highest = 0;
#pragma unroll
    for (int c = 0; c < NG; ++c) highest = max(highest, top[c]);
    if (highest >= 0x7f800000u)     // groups with a NaN: their elements come out as NaN
#pragma unroll
      for (int c = 0; c < NG; ++c) nans |= top[c] >= 0x7f800000u ? 1u << c : 0u;
    __syncwarp();
    int acc[MT][4], eights[NV][4];
    uint32_t vb[NV][2];
#pragma unroll
    for (int nv = 0; nv < NV; ++nv) {
      uint2 v = make_uint2(0, 0);
      if (NG % GT == 0 || g < NG * VC)
        v = *reinterpret_cast<const uint2*>(digits + (nv * 8 + g) * 32 + t * 8);
      vb[nv][0] = v.x;
      vb[nv][1] = v.y;
      mma<false>(eights[nv], kEight, kEightHigh, kEight, kEightHigh, vb[nv]);
    }
    __syncwarp();
#pragma unroll
    for (int c = 0; c < VW; ++c) {
      uint32_t x[2][4];                               // byte j of four keys
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t w[4] = {vw[4 * i][c], vw[4 * i + 1][c], vw[4 * i + 2][c], vw[4 * i + 3][c]};
        transpose_bytes(w, x[i]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        // whole bytes for the high nibbles: 16 times them and the low ones, whose sum is
        // there too
        mma<false>(acc[4 * c + j], x[0][j] & kLow, x[0][j], x[1][j] & kLow, x[1][j],
                   vb[(2 * c + j / 2) / GT]);
    }
    // the columns of this lane belong to one group of each set
#pragma unroll
    for (int nv = 0; nv < NV; ++nv) {
      const int off = eights[nv][0] + eights[nv][1] * 256, off16 = eights[nv][2] + eights[nv][3] * 256;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        int lo = 0, hi = 0;
#pragma unroll
        for (int o = 0; o < GT; ++o) {
          const int mt = 2 * (nv * GT + o) + j;
          if (mt < MT) {
            const int(&a)[4] = acc[mt < MT ? mt : 0];
            lo = owner == o ? a[0] + a[1] * 256 : lo;
            hi = owner == o ? a[2] + a[3] * 256 : hi;
          }
        }
        total[nv][j][0] = fmaf((float)(lo - off), down[nv], total[nv][j][0] * corr);
        total[nv][j][1] = fmaf((float)(hi - lo - off16), down[nv] * 0.0625f, total[nv][j][1] * corr);
      }
    }
  }

  // ---- the warps of a pair ----
#pragma unroll
  for (int nv = 0; nv < NV; ++nv) {
    if (nans && ((nans >> (nv * GT + owner)) & 1u))
#pragma unroll
      for (int j = 0; j < 4; ++j) (&total[nv][0][0])[j] = __uint_as_float(0x7fffffffu);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float v = total[nv][j][r];
        if constexpr (VC == 4)                        // digits 2 and 3 are with the odd lanes
          v = fmaf(__shfl_xor_sync(0xffffffffu, v, 1), 65536.f, v);
        const int gr = nv * GT + owner;
        if (gr < NG && (VC == 2 || (t & 1) == 0))
          s_buf[warp][gr * kGroup + j * 16 + r * 8 + g] = __float_as_uint(v);
      }
  }
  const float l_run = warp_sum(l_lane);
  if (SPLIT && lane == 0) {
    s_ml[warp][0] = m_run;
    s_ml[warp][1] = l_run;
  }
  if constexpr (SPLIT) __syncthreads(); else __syncwarp();
  if (sub == 0 && live) {
  float ref = m_run == -INFINITY ? 0.f : m_run, sum = l_run;
  constexpr int PL = D / 32;                          // elements per lane
  float out[PL];
  if constexpr (SPLIT) {
    float mx = -INFINITY;
    for (int i = 0; i < wpp; ++i) mx = fmaxf(mx, s_ml[warp + i][0]);
    ref = mx == -INFINITY ? 0.f : mx;
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < PL; ++i) out[i] = 0.f;
    for (int i = 0; i < wpp; ++i) {
      const float f = ex2(s_ml[warp + i][0] - ref);
      sum = fmaf(s_ml[warp + i][1], f, sum);
#pragma unroll
      for (int e = 0; e < PL; ++e)
        out[e] = fmaf(__uint_as_float(s_buf[warp + i][lane * PL + e]), f, out[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < PL; ++e) out[e] = __uint_as_float(s_buf[warp][lane * PL + e]);
  }
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(sum));
  if (sum == 0.f) inv = 0.f;
  if constexpr (VC == 2) inv *= kGrow;
  T* o = static_cast<T*>(const_cast<void*>(p.o.data)) + b * p.o.sb + my_h * p.o.sh +
         (int64_t)my_l * p.o.ss + lane * PL;
  struct alignas(PL * sizeof(T) < 16 ? PL * sizeof(T) : 16) Pack { T v[PL]; } pack;
#pragma unroll
  for (int e = 0; e < PL; ++e) pack.v[e] = from_f32<T>(out[e] * inv);
  *reinterpret_cast<Pack*>(o) = pack;
  if (lane == 0) p.lse[((int64_t)b * p.Hq + my_h) * p.span.L + my_l] = ref + log2f(sum);
  }
  __syncwarp();                                      // the buffer holds a query next
  }
}

}  // namespace cache4
}  // namespace esa
