// Weights in 4 bits (esa_int4.cuh, groups of 32, 64 or 128 along the input axis)
// and the product y = x W^T with few rows x.
//
// The product reads N K / 2 bytes of codes for 2 M N K operations: with few rows
// it is bound by that stream, so codes must reach the arithmetic in few
// instructions.  The arithmetic is mma.sync m16n8k16: 16 weight rows as A, 8
// columns (rows of x) as B, float32 sums.  Codes are integers of 4 bits and
// exact in bf16 and fp16, so every product is exact; the sum of a group is
// multiplied by its scale in float32.  (A tcgen05 product would need the codes
// expanded through shared memory first, for tiles of 128 weight rows by as few
// as 8 columns.)  float32 rows of x are split into three bf16 parts (8 bits
// each, exact), three columns whose sums are added at the end.
//
// Layout, made once by quantize_kernel: tiles of 16 weight rows x 64 inputs in
// 512 bytes, 16 per lane (one load), tiles of a row side by side.  Lane 4 g + t
// holds rows g and g + 8, inputs t * 8 .. + 8 of each half of 32; word (half, s)
// holds inputs t * 8 + 4 s + {0, 1, 2, 3} of both rows as the four A registers
// of one mma: nibble j is the low and nibble j + 4 the high element of register
// j.  The same inputs of x are 16 contiguous bytes, so B needs no shared
// memory.  One AND/OR per register makes 128 + n (bf16) or 1024 + n (fp16), one
// subtraction the code.
#pragma once
#include <cooperative_groups.h>

#include "esa_int4.cuh"

namespace esa {
namespace w4 {

constexpr int kTileRows = 16, kBlockK = 64, kBlockBytes = 512;

// ---------------------------------------------------------------------------
// Weights -> codes and scales, and back.  CTA = one tile of rows x 128 inputs;
// thread = 8 inputs of one row.
// ---------------------------------------------------------------------------
struct Packed {
  uint8_t* codes;             // [tiles][blocks][512]
  __nv_bfloat16* scales;      // [tiles][groups][16]
  int N, K, group;
  int tiles, blocks, groups;  // of 16 rows, of 64 inputs, of `group` inputs
};

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
  const int64_t tile = blockIdx.y;
  const int row = (int)(tile * kTileRows) + r;
  const int k = (int)blockIdx.x * 128 + part * 8;
  float f[8];
  load8(w + (int64_t)row * p.K + k, row < p.N, k, p.K, f);
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, int4::abs_bits(f[e]));
  for (int o = 1; o < p.group / 8; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float s = int4::group_scale(top), inv = 1.f / s;
  const int g = k / p.group;
  if (part % (p.group / 8) == 0 && g < p.groups)
    p.scales[(tile * p.groups + g) * kTileRows + r] = __float2bfloat16_rn(s);
  const int shift = r >= 8 ? 4 : 0;                  // registers 1 and 3 hold rows 8 .. 15
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t c[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) c[e] = int4::code_of(f[4 * i + e], s, inv);
    s_words[threadIdx.x][i] = (c[0] | c[1] << 16 | c[2] << 8 | c[3] << 24) << shift;
  }
  __syncthreads();
  const int block = (int)blockIdx.x * 2 + (part >> 3);
  if (r >= 8 || block >= p.blocks) return;
  const int lane = (r << 2) | (part & 3), half = (part >> 2) & 1;
  uint2 out;
  out.x = s_words[threadIdx.x][0] | s_words[threadIdx.x + 128][0];
  out.y = s_words[threadIdx.x][1] | s_words[threadIdx.x + 128][1];
  *reinterpret_cast<uint2*>(p.codes + (tile * p.blocks + block) * kBlockBytes + lane * 16 +
                            half * 8) = out;
}

template <typename T>
__global__ void __launch_bounds__(kPackThreads)
dequantize_kernel(const Packed p, T* w) {
  const int r = threadIdx.x >> 4, part = threadIdx.x & 15;
  const int64_t tile = blockIdx.y;
  const int row = (int)(tile * kTileRows) + r;
  const int k = (int)blockIdx.x * 128 + part * 8;
  if (row >= p.N || k >= p.K) return;
  const int block = (int)blockIdx.x * 2 + (part >> 3);
  const int lane = ((r & 7) << 2) | (part & 3), half = (part >> 2) & 1;
  const uint2 v = __ldg(reinterpret_cast<const uint2*>(
      p.codes + (tile * p.blocks + block) * kBlockBytes + lane * 16 + half * 8));
  const float s = __bfloat162float(p.scales[(tile * p.groups + k / p.group) * kTileRows + r]);
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

template <typename H>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<H, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The four A registers of a word of codes.
template <typename H>
__device__ __forceinline__ void expand(uint32_t w, uint32_t (&a)[4]) {
  constexpr bool kHalf = std::is_same<H, __half>::value;
  constexpr uint32_t kOne = kHalf ? 0x64006400u : 0x43004300u;       // 1024 or 128, twice
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t v = ((w >> (4 * j)) & 0x000f000fu) | kOne;
    if constexpr (kHalf) {
      const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&v), __float2half2_rn(1032.f));
      a[j] = *reinterpret_cast<const uint32_t*>(&d);
    } else {
      const __nv_bfloat162 d =
          __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), __float2bfloat162_rn(136.f));
      a[j] = *reinterpret_cast<const uint32_t*>(&d);
    }
  }
}

// Eight inputs of one column as four B words: x itself, or part `part` of the
// float32 values cut into pieces of 8 significant bits.  (An infinity is all in
// the first part.)
template <typename T>
__device__ __forceinline__ uint4 column8(const T* x, int k, int K, bool in, int part) {
  if constexpr (sizeof(T) == 2) {
    return in && k < K ? ldg16(x + k) : make_uint4(0, 0, 0, 0);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint4 v = in && k + 4 * h < K ? ldg16(x + k + 4 * h) : make_uint4(0, 0, 0, 0);
      const uint32_t u[4] = {v.x, v.y, v.z, v.w};
      uint32_t b[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float r = __uint_as_float(u[e]);
        const bool finite = (u[e] & 0x7f800000u) != 0x7f800000u;
        b[e] = u[e];
        if (part > 0) {
          r -= __uint_as_float(u[e] & 0xffff0000u);
          if (part > 1) r -= __uint_as_float(__float_as_uint(r) & 0xffff0000u);
          b[e] = finite ? __float_as_uint(r) : 0u;
        }
      }
      w[2 * h] = __byte_perm(b[0], b[1], 0x7632);
      w[2 * h + 1] = __byte_perm(b[2], b[3], 0x7632);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <typename T> struct LinearParams {
  const T* x;
  T* y;
  const uint8_t* codes;
  const __nv_bfloat16* scales;
  int M, N, K, group;
  int tiles, blocks, groups;
};

constexpr int kWarps = 8;

// CTA = RT * WR tiles of weight rows x NT * 8 columns; its 8 warps are WR groups
// of rows times WK = 8 / WR parts of K.  A cluster of CTAs along x splits K
// further; the sums are joined in a fixed order.
template <typename T, int NT, int RT, int WR>
__global__ void __launch_bounds__(kWarps * 32)
linear_kernel(const LinearParams<T> p) {
  namespace cg = cooperative_groups;
  using H = typename Operand<T>::Half;
  constexpr int P = Operand<T>::kParts;
  constexpr int WK = kWarps / WR;
  constexpr int kTokens = NT * 8 / P;                  // rows of x per CTA
  constexpr int kRows = RT * WR * kTileRows, kCols = NT * 8;
  __shared__ float s_part[WK][kRows][kCols + 1];
  const cg::cluster_group cluster = cg::this_cluster();
  const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int wr = warp % WR, wk = warp / WR;
  const int g = lane >> 2, t = lane & 3;
  const int tile0 = (int)(blockIdx.x / ctas) * RT * WR + wr * RT;
  const int m0 = (int)blockIdx.y * kTokens;

  // this warp's blocks of K: an even split over the cluster's ctas * WK parts, in
  // whole pairs so that a group of 128 has one owner
  const int pairs = (p.blocks + 1) / 2, share = ctas * WK, me = rank * WK + wk;
  const int b0 = 2 * (int)((int64_t)pairs * me / share);
  const int b1 = min(p.blocks, 2 * (int)((int64_t)pairs * (me + 1) / share));

  float acc[RT][NT][4];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[r][n][i] = 0.f;

  const T* xc[NT];
  bool in[NT];
  int part[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int c = n * 8 + g, token = c / P;
    part[n] = c % P;
    in[n] = token < kTokens && m0 + token < p.M;
    xc[n] = p.x + (int64_t)(in[n] ? m0 + token : 0) * p.K;
  }

  constexpr int U = RT * NT >= 8 ? 2 : 4;              // blocks in flight
  for (int b = b0; b < b1; b += U) {
    uint4 codes[U][RT];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const bool ok = b + u < b1 && tile0 + r < p.tiles;
        codes[u][r] = ok ? ldg16_stream(p.codes + ((int64_t)(tile0 + r) * p.blocks + b + u) * kBlockBytes + lane * 16)
                         : make_uint4(0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u);
      }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (b + u >= b1) break;
      float sum[RT][NT][4];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int k = (b + u) * kBlockK + half * 32;
        uint4 xb[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) xb[n] = column8(xc[n], k + t * 8, p.K, in[n], part[n]);
        const bool fresh = half == 0 || p.group == 32;
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          uint32_t a0[4], a1[4];
          expand<H>(half ? codes[u][r].z : codes[u][r].x, a0);
          expand<H>(half ? codes[u][r].w : codes[u][r].y, a1);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if (fresh)
#pragma unroll
              for (int i = 0; i < 4; ++i) sum[r][n][i] = 0.f;
            mma<H>(sum[r][n], a0, xb[n].x, xb[n].y);
            mma<H>(sum[r][n], a1, xb[n].z, xb[n].w);
          }
        }
        if (half == 1 || p.group == 32) {
          const int gi = k / p.group;
#pragma unroll
          for (int r = 0; r < RT; ++r) {
            if (tile0 + r >= p.tiles || gi >= p.groups) break;
            const __nv_bfloat16* s = p.scales + ((int64_t)(tile0 + r) * p.groups + gi) * kTileRows + g;
            const float lo = __bfloat162float(s[0]), hi = __bfloat162float(s[8]);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              acc[r][n][0] = fmaf(lo, sum[r][n][0], acc[r][n][0]);
              acc[r][n][1] = fmaf(lo, sum[r][n][1], acc[r][n][1]);
              acc[r][n][2] = fmaf(hi, sum[r][n][2], acc[r][n][2]);
              acc[r][n][3] = fmaf(hi, sum[r][n][3], acc[r][n][3]);
            }
          }
        }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        s_part[wk][(wr * RT + r) * kTileRows + g + (i >> 1) * 8][n * 8 + 2 * t + (i & 1)] = acc[r][n][i];
  if (ctas > 1) cluster.sync(); else __syncthreads();
  // outputs of the CTA group, split over the cluster; neighbouring threads write
  // neighbouring weight rows of one row of y
  const int row0 = (int)(blockIdx.x / ctas) * kRows;
  const int tokens = min(kTokens, p.M - m0);
  for (int i = rank * kWarps * 32 + threadIdx.x; i < tokens * kRows; i += ctas * kWarps * 32) {
    const int token = i / kRows, row = i % kRows;
    if (row0 + row >= p.N) continue;
    float sum = 0.f;
    for (int c = 0; c < ctas; ++c) {
      const float* base = ctas > 1 ? cluster.map_shared_rank(&s_part[0][0][0], c) : &s_part[0][0][0];
#pragma unroll
      for (int w = 0; w < WK; ++w)
#pragma unroll
        for (int q = 0; q < P; ++q) sum += base[(w * kRows + row) * (kCols + 1) + token * P + q];
    }
    p.y[(int64_t)(m0 + token) * p.N + row0 + row] = from_f32<T>(sum);
  }
  if (ctas > 1) cluster.sync();      // this CTA's sums are read by the others
}

}  // namespace w4
}  // namespace esa
