// Token embedding: lookup with a scale, and the weight gradient by sorted tokens.
//
//   out[r]  = scale * W[id_r]                                (one rounding)
//   dW[v]   = scale * sum over r with id_r = v of dy[r]        (float32 sums)
//
// Both move rows and do almost no arithmetic: they are bound by HBM.  The
// gradient sums the rows of each token in a fixed order without atomics, so
// it is the same in every run; its rows of tokens that do not occur are zero.
#pragma once
#include "esa_common.cuh"

namespace esa {
namespace embed {

constexpr int kErrTokenRange = 16;   // ESA_DEVERR_TOKEN_RANGE

struct Ids {
  const void* p;
  int wide;     // 1: int64 ids, 0: int32 ids
  __device__ __forceinline__ int64_t get(int64_t i) const {
    return wide ? __ldg(static_cast<const long long*>(p) + i)
                : (int64_t)__ldg(static_cast<const int*>(p) + i);
  }
};

// ---------------------------------------------------------------------------
// Lookup.  The output is cut into runs of kLookupThreads * kLookupUnroll
// 16-byte vectors, one CTA each, whatever the row width; a thread's vectors
// are kLookupThreads apart, so every load and store of a warp is contiguous
// within a row.
// ---------------------------------------------------------------------------
constexpr int kLookupThreads = 128;
constexpr int kLookupUnroll = 4;

template <typename T>
__global__ void __launch_bounds__(kLookupThreads)
lookup_kernel(int64_t n, int64_t vocab, uint32_t vpr, Ids ids, const T* __restrict__ w, float scale,
              T* __restrict__ out, int* err) {
  using V = Vec<T>;
  constexpr int E = V::kElems;
  const int64_t total = n * vpr;
  const int64_t base = (int64_t)blockIdx.x * (kLookupThreads * kLookupUnroll);
  const int64_t tok0 = base / vpr;
  const uint32_t rem0 = (uint32_t)(base - tok0 * vpr);
  // vector and token of this thread, then steps of kLookupThreads vectors
  uint32_t dt = (rem0 + threadIdx.x) / vpr, col = rem0 + threadIdx.x - dt * vpr;
  const uint32_t dt_step = kLookupThreads / vpr, col_step = kLookupThreads - dt_step * vpr;
  uint4 v[kLookupUnroll];
#pragma unroll
  for (int u = 0; u < kLookupUnroll; ++u) {
    v[u] = make_uint4(0, 0, 0, 0);
    if (base + u * kLookupThreads + threadIdx.x < total) {
      const int64_t id = ids.get(tok0 + dt);
      if (id >= 0 && id < vocab) {
        v[u] = ldg16(w + (id * vpr + col) * E);
      } else if (col == 0) {
        atomicOr(err, kErrTokenRange);
      }
    }
    dt += dt_step;
    col += col_step;
    if (col >= vpr) {
      col -= vpr;
      ++dt;
    }
  }
#pragma unroll
  for (int u = 0; u < kLookupUnroll; ++u) {
    const int64_t i = base + u * kLookupThreads + threadIdx.x;
    if (i >= total) break;
    if (scale != 1.f) {          // 1 needs no arithmetic
      float f[E];
      V::to_float(v[u], f);
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] *= scale;
      v[u] = V::from_float(f);
    }
    __stcs(reinterpret_cast<uint4*>(out + i * E), v[u]);
  }
}

// ---------------------------------------------------------------------------
// Gradient, few tokens: one launch, no workspace.  A CTA
// owns R <= 32 rows of dW times 32 * NV vectors of the width.  Each warp lists
// the tokens of these rows in a contiguous quarter of the input, in order, and
// sums its own list; what several warps have of a row is added in warp order.
// NV = 4 for wide rows, whose clearing wants long stores (vocabulary 32000 x
// 4096 bf16: with 1024 tokens 50 us, NV = 1 78; with 8 tokens 40 and 41, torch's
// zero_ of dW alone 70), 1 for narrow ones, whose CTAs would be too few.
// ---------------------------------------------------------------------------
constexpr int kDirectMax = 2048;

// Up to how many tokens: against the sort, vocabulary 32000 in bf16, a call with
// 2048 tokens takes 12 and 17 us at width 64, 63 and 60 at 4096, with 1024 50
// and 54 there.  (1024 times the same token, which one CTA per 128 vectors then
// sums, take 109 us at 4096.)
__host__ __device__ constexpr int direct_max(int dim) {
  return dim <= 256 ? kDirectMax : kDirectMax / 2;
}

constexpr int kDirectThreads = 128;
constexpr int kDirectWarps = kDirectThreads / 32;
constexpr int kDirectPerWarp = kDirectMax / kDirectWarps;
constexpr int kDirectLoads = 16;        // loads in flight per thread

template <typename T>
__device__ __forceinline__ void store_scaled(T* dst, const float* acc, float scale) {
  using V = Vec<T>;
  float o[V::kElems];
#pragma unroll
  for (int e = 0; e < V::kElems; ++e) o[e] = acc[e] * scale;
  stg16(dst, V::from_float(o));
}

// Clears the rows of dW in [v0, v0 + rows) whose bit in `which` is set, all of
// their width (whole: by the CTA's threads through the contiguous block, which
// keeps lanes busy on narrow rows) or 32 * NV vectors from vec0 on (a warp a row).
template <typename T, int Threads, int NV>
__device__ __forceinline__ void clear_rows(T* dw, int64_t v0, int rows, uint32_t which,
                                           uint32_t vpr, uint32_t vec0, bool whole) {
  constexpr int E = Vec<T>::kElems;
  T* dst = dw + v0 * vpr * E;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  if (whole) {
    for (uint32_t i = threadIdx.x; i < rows * vpr; i += Threads)
      if (which >> (i / vpr) & 1) stg16(dst + (int64_t)i * E, zero);
  } else {
    const uint32_t vec = vec0 + (threadIdx.x & 31);
    for (int r = threadIdx.x >> 5; r < rows; r += Threads / 32) {
      if (!(which >> r & 1)) continue;
#pragma unroll
      for (int v = 0; v < NV; ++v)
        if (vec + v * 32 < vpr) stg16(dst + ((int64_t)r * vpr + vec + v * 32) * E, zero);
    }
  }
}

// acc += the rows of a warp's list that belong to row r, in order; lane's
// vectors are vec, vec + 32, ... below vpr.
template <typename T, int NV>
__device__ __forceinline__ void add_listed(const uint32_t* list, int count, int r,
                                           const T* __restrict__ dy, uint32_t vpr, uint32_t vec,
                                           float (&acc)[NV][Vec<T>::kElems]) {
  using V = Vec<T>;
  constexpr int E = V::kElems, U = kDirectLoads / NV;
  const int lane = threadIdx.x & 31;
  for (int j0 = 0; j0 < count; j0 += 32) {
    const uint32_t it = j0 + lane < count ? list[j0 + lane] : 0xffffffffu;
    uint32_t m = __ballot_sync(0xffffffffu, (it >> 16) == (uint32_t)r);
    while (m) {
      uint4 x[U][NV];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const T* src = nullptr;
        if (m) {
          const uint32_t row = __shfl_sync(0xffffffffu, it, __ffs(m) - 1) & 0xffffu;
          m &= m - 1;
          src = dy + ((int64_t)row * vpr + vec) * E;
        }
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          x[u][v] = make_uint4(0, 0, 0, 0);
          if (src && vec + v * 32 < vpr) x[u][v] = ldg16_stream(src + v * 32 * E);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          float f[E];
          V::to_float(x[u][v], f);
#pragma unroll
          for (int e = 0; e < E; ++e) acc[v][e] += f[e];
        }
      }
    }
  }
}

template <typename T, int NV>
__global__ void __launch_bounds__(kDirectThreads)
grad_direct_kernel(int n, int64_t vocab, int R, uint32_t vpr, Ids ids, const T* __restrict__ dy,
                   float scale, int64_t pad, T* __restrict__ dw, int* err) {
  using V = Vec<T>;
  constexpr int E = V::kElems;
  __shared__ uint32_t list[kDirectWarps][kDirectPerWarp];   // (row of dW - v0) << 16 | token
  __shared__ uint32_t present[kDirectWarps];                // rows of dW a warp has tokens of
  __shared__ float part[kDirectWarps][NV * E][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t v0 = (int64_t)blockIdx.x * R;
  const int per_warp = (n + kDirectWarps - 1) / kDirectWarps;
  int count = 0;
  uint32_t rows_seen = 0;
  for (int i0 = 0; i0 < per_warp; i0 += 32) {
    const int i = warp * per_warp + i0 + lane;
    const bool in = i0 + lane < per_warp && i < n;
    const int64_t id = in ? ids.get(i) : -1;
    if (in && (id < 0 || id >= vocab) && blockIdx.x == 0 && blockIdx.y == 0)
      atomicOr(err, kErrTokenRange);
    const bool mine = in && id >= v0 && id < v0 + R && id < vocab && id != pad;
    const uint32_t m = __ballot_sync(0xffffffffu, mine);
    if (mine) {
      list[warp][count + __popc(m & ((1u << lane) - 1))] = (uint32_t)(id - v0) << 16 | (uint32_t)i;
      rows_seen |= 1u << (int)(id - v0);
    }
    count += __popc(m);
  }
  rows_seen = __reduce_or_sync(0xffffffffu, rows_seen);
  if (lane == 0) present[warp] = rows_seen;
  __syncthreads();
  uint32_t any = 0, several = 0;
#pragma unroll
  for (int w = 0; w < kDirectWarps; ++w) {
    several |= any & present[w];
    any |= present[w];
  }
  const uint32_t vec = blockIdx.y * (32 * NV) + lane;
  clear_rows<T, kDirectThreads, NV>(dw, v0, (int)(vocab - v0 < R ? vocab - v0 : R), ~any, vpr,
                                    blockIdx.y * (32 * NV), gridDim.y == 1);
  // rows that this warp has alone
  for (uint32_t own = rows_seen & ~several; own; own &= own - 1) {
    const int r = __ffs(own) - 1;
    float acc[NV][E] = {};
    add_listed<T, NV>(list[warp], count, r, dy, vpr, vec, acc);
#pragma unroll
    for (int v = 0; v < NV; ++v)
      if (vec + v * 32 < vpr)
        store_scaled<T>(dw + ((v0 + r) * vpr + vec + v * 32) * E, acc[v], scale);
  }
  while (several) {
    const int r = __ffs(several) - 1;
    several &= several - 1;
    float acc[NV][E] = {};
    if (rows_seen >> r & 1) add_listed<T, NV>(list[warp], count, r, dy, vpr, vec, acc);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
#pragma unroll
      for (int e = 0; e < E; ++e) part[warp][v * E + e][lane] = acc[v][e];
    }
    __syncthreads();
    // a warp adds up every kDirectWarps-th group of 32 vectors
    for (int v = warp; v < NV; v += kDirectWarps) {
      float sum[E] = {};
#pragma unroll
      for (int w = 0; w < kDirectWarps; ++w) {
#pragma unroll
        for (int e = 0; e < E; ++e) sum[e] += part[w][v * E + e][lane];
      }
      if (vec + v * 32 < vpr)
        store_scaled<T>(dw + ((v0 + r) * vpr + vec + v * 32) * E, sum, scale);
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// Gradient, many tokens.  The (token, row) pairs are sorted by token with a
// stable radix sort (digits of up to 9 bits, low digit first: a histogram and
// a scatter launch per digit), then the sorted list is cut into pieces of
// P pairs that are summed independently.  A run of one token of at most P
// pairs belongs to the piece it starts in; a longer one is cut at the piece
// borders into float32 partial sums, which a last launch adds in order, so no
// CTA's share grows with a token's frequency.
// Tokens that are padding or out of range get the key `vocab` and sort last.
// ---------------------------------------------------------------------------
constexpr int kRadixBits = 9;
constexpr int kRadix = 1 << kRadixBits;
constexpr int kSortThreads = 512;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortItems = 2;
constexpr int kSortTile = kSortThreads * kSortItems;   // keys of a CTA's inner step
constexpr int kSortTiles = 128;       // with more keys than fill them, longer tiles first
constexpr int kSortMaxTiles = 512;    // rows of the histogram table

// Pairs per piece: 64, so that partial sums are few; less for narrow rows and
// fewer tokens, whose time is a piece's chain of loads.  Vocabulary 32000 in
// bf16, P = 16 / 32 / 64: 8192 x 4096 73 / 76 / 80 us, 32768 x 1024 43 / 44 /
// 50, 65536 x 1024 62 / 58 / 61, 131072 x 4096 288 / 256 / 247; 8192 x 64 (with a
// warp per piece) 22 against 32 with 64.
__host__ __device__ constexpr bool narrow_rows(int dim) { return dim <= 256; }
__host__ __device__ constexpr int piece_len(int64_t n, int dim) {
  return narrow_rows(dim) || n <= 8192 ? 16 : n <= 65536 ? 32 : 64;
}
constexpr int kGradUnroll = 8;          // rows in flight per thread

// Key of token i in the first pass.
__device__ __forceinline__ uint32_t token_key(const Ids& ids, int64_t i, int64_t vocab, int64_t pad,
                                              int* err) {
  const int64_t id = ids.get(i);
  if (id < 0 || id >= vocab) {
    if (err) atomicOr(err, kErrTokenRange);
    return (uint32_t)vocab;
  }
  return id == pad ? (uint32_t)vocab : (uint32_t)id;
}

struct SortPass {
  int64_t n, vocab, pad;
  Ids ids;                    // first pass: the tokens; later passes: keys / rows
  const uint32_t* keys;       // nullptr in the first pass
  const uint32_t* rows;
  int shift, bits;
  int tile;                   // keys per CTA, a multiple of kSortTile
  uint32_t* hist;             // [gridDim.x][kRadix]
  uint32_t* out_keys;
  uint32_t* out_rows;
  int* counter;               // of the long runs found later; reset in the first pass
  int* err;
};

// hist[tile][digit] of one pass.
__global__ void __launch_bounds__(kSortThreads) sort_hist_kernel(SortPass p) {
  __shared__ uint32_t h[kRadix];
  cudaTriggerProgrammaticLaunchCompletion();   // the next launch may take free SMs
  for (int i = threadIdx.x; i < kRadix; i += kSortThreads) h[i] = 0;
  cudaGridDependencySynchronize();
  if (!p.keys && blockIdx.x == 0 && threadIdx.x == 0) *p.counter = 0;
  __syncthreads();
  const int64_t lo = (int64_t)blockIdx.x * p.tile;
  const int64_t hi = lo + p.tile < p.n ? lo + p.tile : p.n;
  const uint32_t mask = (1u << p.bits) - 1;
  for (int64_t i = lo + threadIdx.x; i < hi; i += kSortThreads) {
    const uint32_t key = p.keys ? p.keys[i] : token_key(p.ids, i, p.vocab, p.pad, p.err);
    atomicAdd(&h[(key >> p.shift) & mask], 1u);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kRadix; i += kSortThreads)
    p.hist[(int64_t)blockIdx.x * kRadix + i] = h[i];
}

// Stable scatter of one pass: a warp ranks its contiguous keys round by round
// (equal digits of a round by lane), warps and CTAs follow in order.
__global__ void __launch_bounds__(kSortThreads) sort_scatter_kernel(SortPass p) {
  // of a warp's keys, then their places; cleared 16 bytes at a time
  __shared__ __align__(16) uint32_t cnt[kSortWarps][kRadix];
  __shared__ uint32_t wsum[kSortWarps];
  static_assert(kRadix == kSortThreads, "a thread per digit");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, digit = threadIdx.x;
  cudaTriggerProgrammaticLaunchCompletion();
  auto clear = [&] {
    for (int i = threadIdx.x; i < kSortWarps * kRadix / 4; i += kSortThreads)
      reinterpret_cast<uint4*>(&cnt[0][0])[i] = make_uint4(0, 0, 0, 0);
  };
  clear();
  cudaGridDependencySynchronize();
  const uint32_t mask = (1u << p.bits) - 1;
  const int64_t lo = (int64_t)blockIdx.x * p.tile;
  const int64_t hi = lo + p.tile < p.n ? lo + p.tile : p.n;
  uint32_t key[kSortItems], row[kSortItems], rank[kSortItems];
  auto load = [&](int64_t t0) {
#pragma unroll
    for (int r = 0; r < kSortItems; ++r) {
      const int64_t i = t0 + warp * (32 * kSortItems) + r * 32 + lane;
      key[r] = row[r] = 0;
      if (i < hi) {
        key[r] = p.keys ? p.keys[i] : token_key(p.ids, i, p.vocab, p.pad, nullptr);
        row[r] = p.keys ? p.rows[i] : (uint32_t)i;
      }
    }
  };
  load(lo);                                         // on their way during the sums
  uint32_t tot = 0, before = 0;
  const uint32_t* h = p.hist + digit;
  for (int k0 = 0; k0 < (int)gridDim.x; k0 += 32) {
    uint32_t x[32];
#pragma unroll
    for (int u = 0; u < 32; ++u)
      x[u] = k0 + u < (int)gridDim.x ? h[(int64_t)(k0 + u) * kRadix] : 0;
#pragma unroll
    for (int u = 0; u < 32; ++u) {
      tot += x[u];
      if (k0 + u < (int)blockIdx.x) before += x[u];
    }
  }
  uint32_t incl = tot;                              // inclusive scan over digits
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) wsum[warp] = incl;
  __syncthreads();
  uint32_t base = incl - tot + before;              // next output slot of this digit
  for (int w = 0; w < warp; ++w) base += wsum[w];
  for (int64_t t0 = lo; t0 < hi; t0 += kSortTile) {
#pragma unroll
    for (int r = 0; r < kSortItems; ++r) {
      const bool in = t0 + warp * (32 * kSortItems) + r * 32 + lane < hi;
      const uint32_t d = in ? (key[r] >> p.shift) & mask : kRadix;   // kRadix: no key
      const uint32_t same = __match_any_sync(0xffffffffu, d);
      const int before_me = __popc(same & ((1u << lane) - 1));
      if (in) rank[r] = cnt[warp][d] + before_me;
      __syncwarp();
      if (in && before_me == 0) cnt[warp][d] += __popc(same);
      __syncwarp();
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) {
      const uint32_t x = cnt[w][digit];
      cnt[w][digit] = base;
      base += x;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kSortItems; ++r) {
      if (t0 + warp * (32 * kSortItems) + r * 32 + lane < hi) {
        const uint32_t pos = cnt[warp][(key[r] >> p.shift) & mask] + rank[r];
        p.out_keys[pos] = key[r];
        p.out_rows[pos] = row[r];
      }
    }
    if (t0 + kSortTile < hi) {
      load(t0 + kSortTile);
      __syncthreads();
      clear();
      __syncthreads();
    }
  }
}

// The whole sort in one launch of one CTA for up to kSmallMax keys: the same
// passes (digits of up to 8 bits) with keys, rows and counts in shared memory.
// It saves three launches, but its one CTA takes longer with every key.  A
// gradient call (32000 x 1024, bf16) with this and with the general sort, in a
// graph: 24 and 28 us with 1025 keys, 29 and 30 with 2048, 31 and 31 with 2560,
// 37 and 31 with 4096; called singly 37 and 44, 42 and 46, 45 and 46, 50 and 46.
constexpr int kSmallThreads = 1024;
constexpr int kSmallMax = 2560;
constexpr int kSmallItems = (kSmallMax + kSmallThreads - 1) / kSmallThreads;
constexpr int kSmallBits = 8;

struct SmallSort {
  int64_t vocab, pad;
  Ids ids;
  int n, passes, bits;
  uint32_t* out_keys;
  uint32_t* out_rows;
  int* counter;               // of the long runs found later; reset here
  int* err;
};

__global__ void __launch_bounds__(kSmallThreads) sort_small_kernel(SmallSort p) {
  constexpr int W = kSmallThreads / 32, R = 1 << kSmallBits;
  __shared__ uint32_t skey[kSmallMax];
  __shared__ uint16_t srow[kSmallMax];
  // of a warp's keys, then their places; cleared two at a time
  __shared__ __align__(4) uint16_t cnt[W][R];
  __shared__ uint32_t wsum[R / 32];
  cudaTriggerProgrammaticLaunchCompletion();
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  const int items = (p.n + kSmallThreads - 1) / kSmallThreads;
  const int first = warp * items * 32 + lane;
  const uint32_t mask = (1u << p.bits) - 1;
  uint32_t key[kSmallItems], row[kSmallItems], ahead[kSmallItems];
#pragma unroll
  for (int r = 0; r < kSmallItems; ++r) {
    const int i = first + r * 32;
    row[r] = i;
    key[r] = r < items && i < p.n ? token_key(p.ids, i, p.vocab, p.pad, p.err) : 0;
  }
  if (t == 0) *p.counter = 0;
  for (int pass = 0; pass < p.passes; ++pass) {
    for (int i = t; i < W * R / 2; i += kSmallThreads)
      reinterpret_cast<uint32_t*>(&cnt[0][0])[i] = 0;
    __syncthreads();
    if (pass) {
#pragma unroll
      for (int r = 0; r < kSmallItems; ++r) {
        const int i = first + r * 32;
        if (r < items && i < p.n) {
          key[r] = skey[i];
          row[r] = srow[i];
        }
      }
    }
#pragma unroll
    for (int r = 0; r < kSmallItems; ++r) {
      if (r < items) {
        const bool in = first + r * 32 < p.n;
        const uint32_t d = in ? (key[r] >> (pass * p.bits)) & mask : R;   // R: no key
        const uint32_t same = __match_any_sync(0xffffffffu, d);
        const int before_me = __popc(same & ((1u << lane) - 1));
        if (in) ahead[r] = cnt[warp][d] + before_me;
        __syncwarp();
        if (in && before_me == 0) cnt[warp][d] += (uint16_t)__popc(same);
        __syncwarp();
      }
    }
    __syncthreads();
    uint32_t sum = 0, incl = 0;
    if (t < R) {                         // keys of the digit, warp by warp
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const uint32_t x = cnt[w][t];
        cnt[w][t] = (uint16_t)sum;
        sum += x;
      }
      incl = sum;                        // then digit by digit
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      if (lane == 31) wsum[warp] = incl;
    }
    __syncthreads();
    if (t < R) {
      uint32_t off = incl - sum;
      for (int w = 0; w < warp; ++w) off += wsum[w];
#pragma unroll
      for (int w = 0; w < W; ++w) cnt[w][t] += (uint16_t)off;
    }
    __syncthreads();
    const bool last = pass + 1 == p.passes;
#pragma unroll
    for (int r = 0; r < kSmallItems; ++r) {
      if (r < items && first + r * 32 < p.n) {
        const uint32_t pos = cnt[warp][(key[r] >> (pass * p.bits)) & mask] + ahead[r];
        if (last) {
          p.out_keys[pos] = key[r];
          p.out_rows[pos] = row[r];
        } else {
          skey[pos] = key[r];
          srow[pos] = (uint16_t)row[r];
        }
      }
    }
    __syncthreads();
  }
}

// First position in [lo, hi) of the sorted keys that is not below `key`.  The
// sorted pairs are read with ordinary loads here and in the kernels below: the
// sort may still be writing them when those kernels start, and loads through
// the read-only path want memory that does not change while a kernel runs.
__device__ __forceinline__ int64_t lower_bound(const uint32_t* keys, int64_t lo, int64_t hi,
                                               uint32_t key) {
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (keys[mid] < key) lo = mid + 1; else hi = mid;
  }
  return lo;
}

struct GradParams {
  int64_t n, vocab;
  uint32_t vpr;               // 16-byte vectors per row
  const uint32_t* keys;       // sorted
  const uint32_t* rows;
  float scale;
  float* part;                // [pieces][2][dim]: head / tail sums of long runs
  int* counter;               // number of long runs
  uint2* owners;              // each long run's first and last piece
  int64_t pieces;
  int piece;                  // pairs per piece
  int zero_blocks;            // items that clear rows of absent tokens
  int ychunks;                // CTAs per item
};

constexpr int kZeroRows = 32;   // rows of dW per clearing CTA

// One CTA of TH threads per item and TH vectors of the width (TH = 32 for narrow
// rows), the CTAs of an item side by side so that a row's parts are read together.  Items are the pieces with the
// clearing of absent rows spread evenly among them: its searches would leave
// HBM idle if they came first.
template <typename T, int P, int TH>
__global__ void __launch_bounds__(TH)
grad_pieces_kernel(GradParams p, const T* __restrict__ dy, T* __restrict__ dw) {
  using V = Vec<T>;
  constexpr int E = V::kElems;
  __shared__ uint32_t skey[3 * P + 1];   // keys around the piece
  __shared__ uint32_t srow[2 * P];       // rows of the piece and the next
  static_assert(TH > P && kZeroRows == 32, "");
  cudaTriggerProgrammaticLaunchCompletion();
  cudaGridDependencySynchronize();
  const int64_t item = blockIdx.x / p.ychunks;
  const uint32_t chunk = (uint32_t)(blockIdx.x - item * p.ychunks);
  const uint32_t vec = chunk * TH + threadIdx.x;
  const bool active = vec < p.vpr;
  const int64_t items = p.pieces + p.zero_blocks;
  const int64_t zeros = item * p.zero_blocks / items;     // clearing items before this one
  if ((item + 1) * p.zero_blocks / items > zeros) {
    const int64_t v0 = zeros * kZeroRows;
    uint32_t absent = 0;
    if (threadIdx.x < 32) {
      const int64_t v = v0 + threadIdx.x;
      bool none_of_it = false;
      if (v < p.vocab) {
        const int64_t at = lower_bound(p.keys, 0, p.n, (uint32_t)v);
        none_of_it = at == p.n || p.keys[at] != (uint32_t)v;
      }
      absent = __ballot_sync(0xffffffffu, none_of_it);
      if (threadIdx.x == 0) srow[0] = absent;
    }
    __syncthreads();
    const int64_t rows = p.vocab - v0 < kZeroRows ? p.vocab - v0 : kZeroRows;
    clear_rows<T, TH, TH / 32>(dw, v0, (int)rows, srow[0], p.vpr, chunk * TH, p.ychunks == 1);
    return;
  }
  const int64_t piece = item - zeros;
  const int64_t a = piece * P;
  const uint32_t none = 0xffffffffu;      // outside the list, or dropped
  for (int i = threadIdx.x; i < 3 * P + 1; i += TH) {
    const int64_t at = a - P + i;
    uint32_t key = at >= 0 && at < p.n ? p.keys[at] : none;
    if (key >= (uint32_t)p.vocab) key = none;
    skey[i] = key;
    if (i >= P && i < 3 * P && at < p.n) srow[i - P] = p.rows[at];
  }
  __syncthreads();
  const uint32_t* key = skey + P;    // key[i]: entry a + i, i in [-P, 2 P]
  if (key[0] == none) return;             // only dropped tokens from here on
  const int t = threadIdx.x;
  const int len = __syncthreads_count(t < P && key[t] != none);
  // entries before and from the piece's first one that share its key (64 + 65 at
  // most are looked at); the same around its last
  const int fb = __syncthreads_count(t < P && key[t - P] == key[0]);
  const int ff = __syncthreads_count(t <= P && key[t] == key[0]);
  const int lb = __syncthreads_count(t < P && key[len - 1 - t] == key[len - 1]);
  const int lf = __syncthreads_count(t < P && key[len + t] == key[len - 1]);
  const bool long_first = fb + ff > P, long_last = lb + lf > P;
  const int i0 = !long_first && fb > 0 ? ff : 0;           // skip a short run begun earlier
  const int i1 = !long_last ? len + lf : len;              // finish a short run begun here
  // a long run at the end that goes on; listed where it starts
  const bool cut = long_last && lf > 0;
  const bool starts = lb < len || key[-1] != key[0];
  if (cut && starts && chunk == 0 && t == 0)
    p.owners[atomicAdd(p.counter, 1)] =
        make_uint2((uint32_t)piece,
                   (uint32_t)((lower_bound(p.keys, a, p.n, key[len - 1] + 1) - 1) / P));
  if (!active) return;
  const int64_t dim = (int64_t)p.vpr * E;
  bool head = long_first && fb > 0;       // the first run's sum is one of several
  float acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  for (int j0 = i0; j0 < i1; j0 += kGradUnroll) {
    uint4 x[kGradUnroll];
#pragma unroll
    for (int u = 0; u < kGradUnroll; ++u)
      if (j0 + u < i1) x[u] = ldg16_stream(dy + ((int64_t)srow[j0 + u] * p.vpr + vec) * E);
#pragma unroll
    for (int u = 0; u < kGradUnroll; ++u) {
      const int j = j0 + u;
      if (j < i1) {
        float f[E];
        V::to_float(x[u], f);
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] += f[e];
        const bool last = j + 1 == i1;
        if (last || key[j + 1] != key[j]) {
          const bool tail = last && cut;
          if (head || tail) {
            float* dst = p.part + (piece * 2 + (head ? 0 : 1)) * dim + (int64_t)vec * E;
#pragma unroll
            for (int e = 0; e < E; e += 4)
              *reinterpret_cast<float4*>(dst + e) =
                  make_float4(acc[e], acc[e + 1], acc[e + 2], acc[e + 3]);
          } else {
            store_scaled<T>(dw + ((int64_t)key[j] * p.vpr + vec) * E, acc, p.scale);
          }
          head = false;
#pragma unroll
          for (int e = 0; e < E; ++e) acc[e] = 0.f;
        }
      }
    }
  }
}

// Joins the partial sums of the long runs.  A task is (run, 512 columns); its
// warps take every kJoinWarps-th partial, then warp 0 adds theirs in order.
constexpr int kJoinWarps = 8;
constexpr int kJoinVecs = 4;                     // float4 per lane
constexpr int kJoinCols = 128 * kJoinVecs;

__device__ __forceinline__ void add4(float4& a, const float4& x) {
  a.x += x.x; a.y += x.y; a.z += x.z; a.w += x.w;
}

template <typename T>
__global__ void __launch_bounds__(kJoinWarps * 32)
grad_join_kernel(GradParams p, T* __restrict__ dw) {
  __shared__ float4 sum[kJoinWarps][kJoinVecs][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t dim = (int64_t)p.vpr * Vec<T>::kElems;
  const int64_t chunks = (dim + kJoinCols - 1) / kJoinCols;
  cudaGridDependencySynchronize();
  const int64_t tasks = (int64_t)*p.counter * chunks;
  for (int64_t t = blockIdx.x; t < tasks; t += gridDim.x) {
    const uint2 run = p.owners[t / chunks];
    const int64_t piece = run.x, last = run.y;
    const int64_t col = (t % chunks) * kJoinCols + lane * 4;
    const uint32_t key = p.keys[(piece + 1) * p.piece - 1];
    float4 a[kJoinVecs];
#pragma unroll
    for (int v = 0; v < kJoinVecs; ++v) a[v] = make_float4(0.f, 0.f, 0.f, 0.f);
    // slot 1 of the piece it starts in, slot 0 of each later one it reaches
#pragma unroll 4
    for (int64_t q = piece + warp; q <= last; q += kJoinWarps) {
      const float* src = p.part + (q * 2 + (q == piece ? 1 : 0)) * dim + col;
#pragma unroll
      for (int v = 0; v < kJoinVecs; ++v)
        if (col + v * 128 < dim) add4(a[v], *reinterpret_cast<const float4*>(src + v * 128));
    }
#pragma unroll
    for (int v = 0; v < kJoinVecs; ++v) sum[warp][v][lane] = a[v];
    __syncthreads();
    if (warp < kJoinVecs) {
      const int64_t c = col + warp * 128;
      float4 o = sum[0][warp][lane];
#pragma unroll
      for (int w = 1; w < kJoinWarps; ++w) add4(o, sum[w][warp][lane]);
      if (c < dim) {
        T* dst = dw + (int64_t)key * dim + c;
        dst[0] = from_f32<T>(o.x * p.scale);
        dst[1] = from_f32<T>(o.y * p.scale);
        dst[2] = from_f32<T>(o.z * p.scale);
        dst[3] = from_f32<T>(o.w * p.scale);
      }
    }
    __syncthreads();
  }
}

}  // namespace embed
}  // namespace esa
