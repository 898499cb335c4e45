// Weights in 4 bits (esa_int4.cuh, groups of 32, 64 or 128 along the input axis)
// and the product y = x W^T with few rows x.
//
// The product reads N K / 2 bytes of codes for 2 M N K operations: with few rows
// it is bound by that stream, so codes must reach the arithmetic in few
// instructions.  The arithmetic is mma.sync m16n8k16: 16 weight rows as A, 8
// columns (rows of x) as B, float32 sums.  Codes are integers of 4 bits and
// exact in bf16 and fp16, so every product is exact; the sum of a group is
// multiplied by its scale in float32.  (A tcgen05 product takes tiles of 128 weight
// rows, whose decoded codes could go from registers to tensor memory, and its
// accumulator would be read once per group for the scale; it was not built.)  float32
// rows of x are split into three bf16 parts (8 bits each, exact down to 2^-133), three
// columns whose sums are added at the end.
//
// Measured (1 x B200, weights from HBM, launches one after the other): 1 x 4096 x
// 12288 in 9.1 us (its bytes alone: 4.0; a copy of an earlier state of the kernel with
// the arithmetic taken out needed 6.8, without x as well 5.8), 32 x 11008 x 4096 in 15.7
// (3.7), where the matrix instructions alone take 5.2 at their measured rate, the reads
// of x from shared memory by every warp for its 16 weight rows 5.0, and a CTA has only
// some six stages of K.  Not taken up: x in fixed
// point against 8-bit integer products, which needs a third of the instructions for
// one row but took as long (the chain of loads bounds it), and loses bits of float32
// rows with a wide range.
//
// Layout, made once by quantize_kernel: 16 weight rows x 128 inputs in 1024 bytes
// (the tiles of a row side by side, padded with zeros to whole tiles), twice 16
// bytes per lane.  Lane 4 g + t holds rows g and g + 8, inputs t * 8 .. + 8 of each
// 32; word (32, s) holds inputs t * 8 + 4 s + {0, 1, 2, 3} of both rows as the four
// A registers of one mma: nibble j is the low and nibble j + 4 the high element of
// register j.  The same inputs of x are 16 contiguous bytes: one load is the B
// operand of two products.  One AND/OR per register makes 128 + n (bf16) or
// 1024 + n (fp16), one subtraction the code.
#pragma once
#include <cooperative_groups.h>

#include "esa_int4.cuh"

namespace esa {
namespace w4 {

constexpr int kTileRows = 16, kTileK = 128, kTileBytes = 1024;

// ---------------------------------------------------------------------------
// Weights -> codes and scales, and back.  CTA = one tile of rows x 128 inputs;
// thread = 8 inputs of one row.
// ---------------------------------------------------------------------------
struct Packed {
  uint8_t* codes;             // [tiles][chunks][1024]
  __nv_bfloat16* scales;      // [tiles][groups][16]: rows 0, 8, 1, 9, ...
  int N, K, group;
  int tiles, chunks, groups;  // of 16 rows, of 128 inputs, chunks * 128 / group
};

// Place of row r of 16 among the scales of a group.
__device__ __forceinline__ int scale_place(int r) { return (r & 7) * 2 + (r >> 3); }

constexpr int kPackThreads = 256;

template <typename T>
__device__ __forceinline__ void load8(const T* p, bool in, int k, int K, float (&f)[8]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint4 v = in && k + 4 * h < K ? ldg16(p + 4 * h) : make_uint4(0, 0, 0, 0);
      Vec<T>::to_float(v, f + 4 * h);
    }
  } else {
    const uint4 v = in && k < K ? ldg16(p) : make_uint4(0, 0, 0, 0);
    Vec<T>::to_float(v, f);
  }
}

template <typename T>
__global__ void __launch_bounds__(kPackThreads)
quantize_kernel(const Packed p, const T* w) {
  __shared__ uint32_t s_words[kPackThreads][2];
  const int r = threadIdx.x >> 4, part = threadIdx.x & 15;
  const int64_t tile = blockIdx.x / (unsigned)p.chunks;
  const int chunk = (int)(blockIdx.x % (unsigned)p.chunks);
  const int row = (int)(tile * kTileRows) + r;
  const int k = chunk * 128 + part * 8;
  float f[8];
  load8(w + (int64_t)row * p.K + k, row < p.N, k, p.K, f);
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, int4::abs_bits(f[e]));
  for (int o = 1; o < p.group / 8; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  float inv;
  const float s = int4::group_scale(top, inv);
  const uint32_t w8 = int4::codes_of<T>(f, s, inv);
  const int g = k / p.group;
  if (part % (p.group / 8) == 0)
    p.scales[(tile * p.groups + g) * kTileRows + scale_place(r)] = __float2bfloat16_rn(s);
  const int shift = r >= 8 ? 4 : 0;                  // registers 1 and 3 hold rows 8 .. 15
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t c = w8 >> (16 * i);
    s_words[threadIdx.x][i] =
        ((c & 15u) | (c >> 4 & 15u) << 16 | (c >> 8 & 15u) << 8 | (c >> 12 & 15u) << 24) << shift;
  }
  __syncthreads();
  if (r >= 8) return;
  const int lane = (r << 2) | (part & 3), half = (part >> 2) & 1;
  uint2 out;
  out.x = s_words[threadIdx.x][0] | s_words[threadIdx.x + 128][0];
  out.y = s_words[threadIdx.x][1] | s_words[threadIdx.x + 128][1];
  *reinterpret_cast<uint2*>(p.codes + (tile * p.chunks + chunk) * kTileBytes +
                            (part >> 3) * 512 + lane * 16 + half * 8) = out;
}

template <typename T>
__global__ void __launch_bounds__(kPackThreads)
dequantize_kernel(const Packed p, T* w) {
  const int r = threadIdx.x >> 4, part = threadIdx.x & 15;
  const int64_t tile = blockIdx.x / (unsigned)p.chunks;
  const int chunk = (int)(blockIdx.x % (unsigned)p.chunks);
  const int row = (int)(tile * kTileRows) + r;
  const int k = chunk * 128 + part * 8;
  if (row >= p.N || k >= p.K) return;
  const int lane = ((r & 7) << 2) | (part & 3), half = (part >> 2) & 1;
  const uint2 v = __ldg(reinterpret_cast<const uint2*>(
      p.codes + (tile * p.chunks + chunk) * kTileBytes + (part >> 3) * 512 + lane * 16 +
      half * 8));
  const float s =
      __bfloat162float(p.scales[(tile * p.groups + k / p.group) * kTileRows + scale_place(r)]);
  const uint32_t words[2] = {v.x >> (r >= 8 ? 4 : 0), v.y >> (r >= 8 ? 4 : 0)};
  float f[8];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    f[4 * i] = int4::decode(words[i], s);
    f[4 * i + 1] = int4::decode(words[i] >> 16, s);
    f[4 * i + 2] = int4::decode(words[i] >> 8, s);
    f[4 * i + 3] = int4::decode(words[i] >> 24, s);
  }
  T* out = w + (int64_t)row * p.K + k;
#pragma unroll
  for (int h = 0; h < 8 / Vec<T>::kElems; ++h)
    if (k + h * Vec<T>::kElems < p.K) stg16(out + h * Vec<T>::kElems, Vec<T>::from_float(f + h * Vec<T>::kElems));
}

// ---------------------------------------------------------------------------
// The product.
// ---------------------------------------------------------------------------
// The 16-bit type of the matrix instruction and the columns a row of x takes.
template <typename T> struct Operand { using Half = T; static constexpr int kParts = 1; };
template <> struct Operand<float> { using Half = __nv_bfloat16; static constexpr int kParts = 3; };

// c = A B + (FRESH ? 0 : c).  Volatile: all lanes of a warp execute it together.
template <typename H, bool FRESH>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
#define ESA_MMA(T)                                                                               \
  if constexpr (FRESH)                                                                           \
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32." T "." T ".f32 {%0,%1,%2,%3}, "         \
                 "{%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"                                    \
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])                                \
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));      \
  else                                                                                           \
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32." T "." T ".f32 {%0,%1,%2,%3}, "         \
                 "{%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"                                        \
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])                                \
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1))
  if constexpr (std::is_same<H, __half>::value) {
    ESA_MMA("f16");
  } else {
    ESA_MMA("bf16");
  }
#undef ESA_MMA
}

// The four A registers of a word of codes.  bf16 has room for a nibble at the low end
// of its 7 bits only: 128 + n, less 136.  fp16 takes nibbles 0 and 1 of its 10 bits
// where they lie: 1024 + n less 1032, (1024 + 16 n) / 16 less 72.
template <typename H>
__device__ __forceinline__ void expand(uint32_t w, uint32_t (&a)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (std::is_same<H, __half>::value) {
      const uint32_t v = int4::and_or(j < 2 ? w : w >> 8, j & 1 ? 0x00f000f0u : 0x000f000fu, 0x64006400u);
      const __half2 h = *reinterpret_cast<const __half2*>(&v);
      const __half2 d = j & 1 ? __hfma2(h, __float2half2_rn(0.0625f), __float2half2_rn(-72.f))
                              : __hadd2(h, __float2half2_rn(-1032.f));
      a[j] = *reinterpret_cast<const uint32_t*>(&d);
    } else {
      const uint32_t v = int4::and_or(w >> (4 * j), 0x000f000fu, 0x43004300u);
      const __nv_bfloat162 d =
          __hadd2(*reinterpret_cast<const __nv_bfloat162*>(&v), __float2bfloat162_rn(-136.f));
      a[j] = *reinterpret_cast<const uint32_t*>(&d);
    }
  }
}

// Part `part` of eight float32 values cut into pieces of 8 significant bits.  (An
// infinity or a NaN is all in the first part; a NaN's set bits may all be among those
// that are cut off, so it gets one that is not.)
__device__ __forceinline__ uint4 cut8(const uint4& lo, const uint4& hi, int part) {
  const uint32_t u[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
  uint32_t b[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    b[e] = (u[e] & 0x7fffffffu) > 0x7f800000u ? u[e] | 0x00400000u : u[e];
    if (part > 0) {
      float r = __uint_as_float(u[e]) - __uint_as_float(u[e] & 0xffff0000u);
      if (part > 1) r -= __uint_as_float(__float_as_uint(r) & 0xffff0000u);
      b[e] = (u[e] & 0x7f800000u) != 0x7f800000u ? __float_as_uint(r) : 0u;
    }
  }
  return make_uint4(__byte_perm(b[0], b[1], 0x7632), __byte_perm(b[2], b[3], 0x7632),
                    __byte_perm(b[4], b[5], 0x7632), __byte_perm(b[6], b[7], 0x7632));
}

template <typename T> struct LinearParams {
  const T* x;
  T* y;
  const uint8_t* codes;
  const __nv_bfloat16* scales;
  int M, N, K;
  int tiles, chunks;
};

__device__ __forceinline__ void copy16_async(uint32_t to, const void* from, bool in = true) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(in ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void wait_copies() {     // all but the last N groups
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A tile of 16 x 128 codes and the scales of its groups, as one lane holds them.
// They come through shared memory, each lane copying what it reads itself: many
// tiles can be on their way without registers, and no barrier is needed.
template <int G> struct Tile {
  static constexpr int kGroups = kTileK / G;
  static constexpr int kBytes = kTileBytes + kGroups * 128;           // in shared memory
  uint4 c[2];
  uint32_t s[kGroups];         // rows g and g + 8
  // Asks for `count` tiles from `tile` on in L2, where a later write of them is seen:
  // this alone may be done before the kernel before has been waited for, which may
  // have made the codes.
  __device__ __forceinline__ static void prefetch(const uint8_t* codes, const __nv_bfloat16* scales,
                                                  int64_t tile, int count) {
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(codes + tile * kTileBytes),
                 "r"(count * kTileBytes) : "memory");
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(scales + tile * (kGroups * 16)),
                 "r"(count * kGroups * 32) : "memory");
  }
  __device__ __forceinline__ static void fetch(uint32_t to, const uint8_t* codes,
                                               const __nv_bfloat16* scales, int64_t tile, int lane) {
    copy16_async(to + lane * 16, codes + tile * kTileBytes + lane * 16);
    copy16_async(to + 512 + lane * 16, codes + tile * kTileBytes + 512 + lane * 16);
#pragma unroll
    for (int i = 0; i < kGroups; ++i)
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to + kTileBytes + i * 128 + lane * 4),
                   "l"(reinterpret_cast<const uint32_t*>(scales) + (tile * kGroups + i) * 8 + (lane >> 2))
                   : "memory");
  }
  __device__ __forceinline__ void take(const unsigned char* from, int lane) {
    c[0] = *reinterpret_cast<const uint4*>(from + lane * 16);
    c[1] = *reinterpret_cast<const uint4*>(from + 512 + lane * 16);
#pragma unroll
    for (int i = 0; i < kGroups; ++i)
      s[i] = *reinterpret_cast<const uint32_t*>(from + kTileBytes + i * 128 + lane * 4);
  }
  __device__ __forceinline__ uint32_t word(int i) const {      // i = quarter of 32 inputs, s
    const uint4& v = c[i >> 2];
    return (i & 3) == 0 ? v.x : (i & 3) == 1 ? v.y : (i & 3) == 2 ? v.z : v.w;
  }
};

// acc += tile times 128 inputs of NT * 8 columns; B of quarter q in xb(q, n).
template <typename H, int G, int NT, typename B>
__device__ __forceinline__ void multiply(const Tile<G>& w, float (&acc)[NT][4], B&& xb) {
  float sum[NT][4];
  uint4 b[2][NT];                                      // the next quarter's B loads run ahead
#pragma unroll
  for (int n = 0; n < NT; ++n) b[0][n] = xb(0, n);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    if (q < 3)
#pragma unroll
      for (int n = 0; n < NT; ++n) b[(q + 1) & 1][n] = xb(q + 1, n);
    uint32_t a0[4], a1[4];
    expand<H>(w.word(2 * q), a0);
    expand<H>(w.word(2 * q + 1), a1);
    // products of the same sum apart from each other
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if ((q * 32) % G == 0) mma<H, true>(sum[n], a0, b[q & 1][n].x, b[q & 1][n].y);
      else mma<H, false>(sum[n], a0, b[q & 1][n].x, b[q & 1][n].y);
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) mma<H, false>(sum[n], a1, b[q & 1][n].z, b[q & 1][n].w);
    if ((q * 32 + 32) % G == 0) {
      const uint32_t s = w.s[q * 32 / G];
      const float lo = __uint_as_float(s << 16), hi = __uint_as_float(s & 0xffff0000u);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        acc[n][0] = fmaf(lo, sum[n][0], acc[n][0]);
        acc[n][1] = fmaf(lo, sum[n][1], acc[n][1]);
        acc[n][2] = fmaf(hi, sum[n][2], acc[n][2]);
        acc[n][3] = fmaf(hi, sum[n][3], acc[n][3]);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Up to 8 rows of a 16-bit type: bound by the stream of codes.  CTA = one tile of 16 weight rows,
// its WK warps share K and join in shared memory.  A warp has kDepth tiles on their
// way.  Before it waits for the kernel before it (which made x, or the codes) it only
// has the first of them brought into L2.
// ---------------------------------------------------------------------------
constexpr int kDepth = 4;

template <typename T, int G, int WK>
__global__ void __launch_bounds__(WK * 32)
vector_kernel(const LinearParams<T> p) {
  static_assert(Operand<T>::kParts == 1, "a column per row of x");
  extern __shared__ __align__(128) unsigned char s_mem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int c0 = (int)((int64_t)p.chunks * warp / WK), c1 = (int)((int64_t)p.chunks * (warp + 1) / WK);
  const int64_t base = (int64_t)blockIdx.x * p.chunks;
  unsigned char* ring = s_mem + warp * (kDepth * Tile<G>::kBytes);
  const uint32_t to = (uint32_t)__cvta_generic_to_shared(ring);
  if (lane == 0 && c0 < c1) Tile<G>::prefetch(p.codes, p.scales, base + c0, min(kDepth, c1 - c0));
  cudaTriggerProgrammaticLaunchCompletion();           // the next kernel may begin like this
  cudaGridDependencySynchronize();
#pragma unroll
  for (int i = 0; i < kDepth; ++i) {
    if (c0 + i < c1) Tile<G>::fetch(to + i * Tile<G>::kBytes, p.codes, p.scales, base + c0 + i, lane);
    commit_copies();
  }
  const bool in = g < p.M;                             // column g: row g of x
  const T* x = p.x + (int64_t)(in ? g : 0) * p.K + t * 8;
  const int left = p.K - t * 8;
  float acc[1][4] = {{0.f, 0.f, 0.f, 0.f}};
  uint4 xb[4];
  auto inputs = [&](int c) {                           // zeros past K
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int k = c * kTileK + q * 32;
      xb[q] = in && k < left ? ld16(x + k) : make_uint4(0, 0, 0, 0);
    }
  };
  if (c0 < c1) inputs(c0);
#pragma unroll 2
  for (int c = c0; c < c1; ++c) {
    wait_copies<kDepth - 1>();
    const int slot = (c - c0) % kDepth;
    Tile<G> w;
    w.take(ring + slot * Tile<G>::kBytes, lane);
    const uint4 now[4] = {xb[0], xb[1], xb[2], xb[3]};
    if (c + 1 < c1) inputs(c + 1);
    multiply<T, G, 1>(w, acc, [&](int q, int) { return now[q]; });
    // the slot's next tile: the products have waited for what this lane read, and
    // nobody else reads it
    if (c + kDepth < c1)
      Tile<G>::fetch(to + slot * Tile<G>::kBytes, p.codes, p.scales, base + c + kDepth, lane);
    commit_copies();
  }
  __syncthreads();                                     // the ring holds the sums now
  float(*part_sums)[8][kTileRows] = reinterpret_cast<float(*)[8][kTileRows]>(s_mem);
#pragma unroll
  for (int i = 0; i < 4; ++i) part_sums[warp][2 * t + (i & 1)][g + (i >> 1) * 8] = acc[0][i];
  __syncthreads();
  const int row = threadIdx.x & 15;
  for (int m = threadIdx.x >> 4; m < p.M; m += WK * 2) {
    if ((int64_t)blockIdx.x * kTileRows + row >= p.N) break;
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < WK; ++k) sum += part_sums[k][m][row];
    p.y[(int64_t)m * p.N + (int64_t)blockIdx.x * kTileRows + row] = from_f32<T>(sum);
  }
}

// ---------------------------------------------------------------------------
// More columns.  CTA = 8 warps, a tile of 16 weight rows each, times NT * 8 columns;
// a cluster of CTAs along x splits K.  The columns' inputs go through shared memory
// for all warps, the codes for the warp that uses them, kStages stages of kStage
// tiles of K in a ring; a column's inputs lie 64 bytes (mod 128) after those of the
// one before, so that the lanes' 16-byte reads meet no bank twice.
// ---------------------------------------------------------------------------
constexpr int kWarps = 8;

template <typename T, int G, int NT> struct Shape {
  static constexpr int kParts = Operand<T>::kParts;
  static constexpr int kTokens = NT * 8 / kParts;        // rows of x per CTA
  static constexpr int kRows = kWarps * kTileRows, kCols = NT * 8;
  // Tiles of K in a stage and stages in the ring, so that two CTAs fit an SM (a third
  // of the speed is lost where one does).
  static constexpr int kStage = NT == 2 ? 2 : 1;
  static constexpr int kStages = NT == 4 ? 5 : 3;
  static constexpr int kPitch = kStage * kTileK * 2 + 64;              // bytes of a column
  static constexpr int kInputBytes = kCols * kPitch;
  static constexpr int kStageBytes = kInputBytes + kWarps * kStage * Tile<G>::kBytes;
  static constexpr int kSumPitch = kRows + 4;            // floats of a column's sums
  static constexpr int kSumBytes = kCols * kSumPitch * 4;
  static constexpr int kShared = kStages * kStageBytes > kSumBytes ? kStages * kStageBytes : kSumBytes;
  static_assert(kShared <= 112 * 1024, "two CTAs per SM");
};

template <typename T, int G, int NT>
__global__ void __launch_bounds__(kWarps * 32, 2)
rows_kernel(const LinearParams<T> p) {
  namespace cg = cooperative_groups;
  using S = Shape<T, G, NT>;
  using H = typename Operand<T>::Half;
  constexpr int P = S::kParts;
  extern __shared__ __align__(128) unsigned char s_mem[];
  const cg::cluster_group cluster = cg::this_cluster();
  const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int tile = (int)(blockIdx.x / ctas) * kWarps + warp;
  const int m0 = (int)blockIdx.y * S::kTokens;
  const int tokens = min(S::kTokens, p.M - m0);
  const int c0 = (int)((int64_t)p.chunks * rank / ctas), c1 = (int)((int64_t)p.chunks * (rank + 1) / ctas);
  // a warp past the last tile computes that one again
  const int64_t base = (int64_t)min(tile, p.tiles - 1) * p.chunks;
  const uint32_t shared = (uint32_t)__cvta_generic_to_shared(s_mem);

  float acc[NT][4];
#pragma unroll
  for (int i = 0; i < NT * 4; ++i) (&acc[0][0])[i] = 0.f;
  auto fetch_codes = [&](int s, int slot) {              // of stage s: chunks c0 + s * kStage ..
#pragma unroll
    for (int i = 0; i < S::kStage; ++i)
      if (c0 + s * S::kStage + i < c1)
        Tile<G>::fetch(shared + slot * S::kStageBytes + S::kInputBytes + (warp * S::kStage + i) * Tile<G>::kBytes,
                       p.codes, p.scales, base + c0 + s * S::kStage + i, lane);
  };
  // 8 inputs of a row of x per thread and step, zeros where there is no row or input
  constexpr int kSteps = S::kStage * 16;
  constexpr int kTokenStep = kWarps * 32 / kSteps;
  const int k8 = threadIdx.x % kSteps, token0 = threadIdx.x / kSteps;
  const T* const x0 = p.x + (int64_t)(m0 + min(token0, tokens - 1)) * p.K + (int64_t)c0 * kTileK + k8 * 8;
  const int left = p.K - c0 * kTileK - k8 * 8;           // inputs of the row from there
  auto fetch_inputs = [&](int s, int slot) {
    unsigned char* buf = s_mem + slot * S::kStageBytes + k8 * 16 + token0 * P * S::kPitch;
    const uint32_t to = shared + slot * S::kStageBytes + k8 * 16 + token0 * S::kPitch;
    const int k = s * S::kStage * kTileK;
    const T* x = x0 + k;
#pragma unroll
    for (int j = 0; j < (S::kTokens + kTokenStep - 1) / kTokenStep; ++j) {
      const bool row = token0 + j * kTokenStep < tokens;
      if constexpr (P == 1) {
        const bool in = row && k < left;
        copy16_async(to + j * kTokenStep * S::kPitch, in ? x : p.x, in);
      } else if (token0 + j * kTokenStep < S::kTokens) {
        const uint4 none = make_uint4(0, 0, 0, 0);
        const uint4 lo = row && k < left ? ld16(x) : none;
        const uint4 hi = row && k + 4 < left ? ld16(x + 4) : none;
#pragma unroll
        for (int q = 0; q < P; ++q)
          *reinterpret_cast<uint4*>(buf + (j * kTokenStep * P + q) * S::kPitch) = cut8(lo, hi, q);
      }
      if (token0 + (j + 1) * kTokenStep < tokens) x += (int64_t)kTokenStep * p.K;
    }
  };
  if constexpr (S::kTokens * P < S::kCols) {             // columns without a row of x
    constexpr int kSpare = (S::kCols - S::kTokens * P) * (S::kPitch / 16);
    for (int i = threadIdx.x; i < S::kStages * kSpare; i += kWarps * 32)
      *reinterpret_cast<uint4*>(s_mem + i / kSpare * S::kStageBytes + S::kTokens * P * S::kPitch +
                                i % kSpare * 16) = make_uint4(0, 0, 0, 0);
  }
  const int stages = (c1 - c0 + S::kStage - 1) / S::kStage;
  // the codes of the first stages are on their way to L2 before x is waited for
  if (lane == 0 && c0 < c1)
    Tile<G>::prefetch(p.codes, p.scales, base + c0, min((S::kStages - 1) * S::kStage, c1 - c0));
  cudaTriggerProgrammaticLaunchCompletion();             // the next kernel may begin like this
  cudaGridDependencySynchronize();
#pragma unroll
  for (int s = 0; s < S::kStages - 1; ++s) {
    fetch_codes(s, s);
    if (s < stages) fetch_inputs(s, s);
    commit_copies();
  }
  int slot = 0;
#pragma unroll 1
  for (int s = 0; s < stages; ++s) {
    wait_copies<S::kStages - 2>();
    __syncthreads();               // stage s has come; the one before it is no longer read
    const int next = slot == 0 ? S::kStages - 1 : slot - 1;
    if (s + S::kStages - 1 < stages) {
      fetch_codes(s + S::kStages - 1, next);
      fetch_inputs(s + S::kStages - 1, next);
    }
    commit_copies();
    const unsigned char* buf = s_mem + slot * S::kStageBytes;
#pragma unroll
    for (int i = 0; i < S::kStage; ++i) {
      if (c0 + s * S::kStage + i >= c1) break;
      Tile<G> w;
      w.take(buf + S::kInputBytes + (warp * S::kStage + i) * Tile<G>::kBytes, lane);
      const unsigned char* xs = buf + g * S::kPitch + i * (kTileK * 2) + t * 16;
      multiply<H, G, NT>(w, acc, [&](int q, int n) {
        return *reinterpret_cast<const uint4*>(xs + n * 8 * S::kPitch + q * 64);
      });
    }
    slot = slot == S::kStages - 1 ? 0 : slot + 1;
  }
  wait_copies<0>();
  __syncthreads();
  // [columns][rows]: neighbouring lanes read neighbouring words of another CTA's sums
  // (one by one they cost the SM-to-SM network a packet each)
  float* sums = reinterpret_cast<float*>(s_mem);
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      sums[(n * 8 + 2 * t + (i & 1)) * S::kSumPitch + warp * kTileRows + g + (i >> 1) * 8] = acc[n][i];
  if (ctas > 1) cluster.sync(); else __syncthreads();
  // the outputs are split over the cluster; neighbouring threads write neighbouring
  // weight rows of one row of y
  const int row0 = (int)(blockIdx.x / ctas) * S::kRows;
  for (int i = rank * kWarps * 32 + threadIdx.x; i < tokens * S::kRows; i += ctas * kWarps * 32) {
    const int token = i / S::kRows, row = i % S::kRows;
    if (row0 + row >= p.N) continue;
    float v[8][P], sum = 0.f;                            // all loads, then the sum in order
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      if (c < ctas) {
        const float* from = ctas > 1 ? cluster.map_shared_rank(sums, c) : sums;
#pragma unroll
        for (int q = 0; q < P; ++q) v[c][q] = from[(token * P + q) * S::kSumPitch + row];
      }
    }
#pragma unroll
    for (int c = 0; c < 8; ++c)
      if (c < ctas)
#pragma unroll
        for (int q = 0; q < P; ++q) sum += v[c][q];
    p.y[(int64_t)(m0 + token) * p.N + row0 + row] = from_f32<T>(sum);
  }
  if (ctas > 1) cluster.sync();      // this CTA's sums are read by the others
}

}  // namespace w4
}  // namespace esa
