// Token embedding: lookup with a scale, and the weight gradient by sorted tokens.
//
//   out[r]  = scale * W[id_r]                                (one rounding)
//   dW[v]   = scale * sum over r ascending, id_r = v, of dy[r]   (float32 sums)
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
  uint4 v[kLookupUnroll];
#pragma unroll
  for (int u = 0; u < kLookupUnroll; ++u) {
    const uint32_t local = rem0 + u * kLookupThreads + threadIdx.x;
    v[u] = make_uint4(0, 0, 0, 0);
    if (base + u * kLookupThreads + threadIdx.x < total) {
      const uint32_t dt = local / vpr;
      const int64_t id = ids.get(tok0 + dt);
      if (id >= 0 && id < vocab) {
        v[u] = ldg16(w + (id * vpr + (local - dt * vpr)) * E);
      } else if (local - dt * vpr == 0) {
        atomicOr(err, kErrTokenRange);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < kLookupUnroll; ++u) {
    const int64_t i = base + u * kLookupThreads + threadIdx.x;
    if (i < total) {
      float f[E];
      V::to_float(v[u], f);
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] *= scale;
      stg16(out + i * E, V::from_float(f));
    }
  }
}

// ---------------------------------------------------------------------------
// Gradient, few tokens (n <= kDirectMax): one launch, no workspace.  A CTA
// owns R rows of dW times 128 vectors of the width; it lists the tokens of
// its rows (in ascending order: each warp lists a contiguous part) and sums
// each row's list.
// ---------------------------------------------------------------------------
constexpr int kGradThreads = 128;
constexpr int kGradWarps = kGradThreads / 32;
constexpr int kDirectMax = 1024;
constexpr int kDirectPerWarp = kDirectMax / kGradWarps;

template <typename T>
__device__ __forceinline__ void store_scaled(T* dst, const float* acc, float scale) {
  using V = Vec<T>;
  float o[V::kElems];
#pragma unroll
  for (int e = 0; e < V::kElems; ++e) o[e] = acc[e] * scale;
  stg16(dst, V::from_float(o));
}

template <typename T>
__global__ void __launch_bounds__(kGradThreads)
grad_direct_kernel(int n, int64_t vocab, int R, uint32_t vpr, Ids ids, const T* __restrict__ dy,
                   float scale, int64_t pad, T* __restrict__ dw, int* err) {
  using V = Vec<T>;
  constexpr int E = V::kElems;
  __shared__ uint32_t list[kGradWarps][kDirectPerWarp];   // (row of dW - v0) << 16 | token
  __shared__ int count[kGradWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t v0 = (int64_t)blockIdx.x * R;
  const int per_warp = (n + kGradWarps - 1) / kGradWarps;
  int c = 0;
  for (int i0 = 0; i0 < per_warp; i0 += 32) {
    const int i = warp * per_warp + i0 + lane;
    const bool in = i0 + lane < per_warp && i < n;
    const int64_t id = in ? ids.get(i) : -1;
    if (in && (id < 0 || id >= vocab) && blockIdx.x == 0 && blockIdx.y == 0)
      atomicOr(err, kErrTokenRange);
    const bool mine = in && id >= v0 && id < v0 + R && id < vocab && id != pad;
    const uint32_t m = __ballot_sync(0xffffffffu, mine);
    if (mine)
      list[warp][c + __popc(m & ((1u << lane) - 1))] = (uint32_t)(id - v0) << 16 | (uint32_t)i;
    c += __popc(m);
  }
  if (lane == 0) count[warp] = c;
  __syncthreads();
  const uint32_t vec = blockIdx.y * kGradThreads + threadIdx.x;
  if (vec >= vpr) return;
  for (int r = 0; r < R && v0 + r < vocab; ++r) {
    float acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
    for (int wi = 0; wi < kGradWarps; ++wi) {
      for (int j = 0; j < count[wi]; ++j) {
        const uint32_t it = list[wi][j];
        if ((int)(it >> 16) != r) continue;
        float f[E];
        V::to_float(ldg16_stream(dy + ((int64_t)(it & 0xffffu) * vpr + vec) * E), f);
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] += f[e];
      }
    }
    store_scaled<T>(dw + ((v0 + r) * vpr + vec) * E, acc, scale);
  }
}

// ---------------------------------------------------------------------------
// Gradient, many tokens.  The (token, row) pairs are sorted by token with a
// stable radix sort (digits of up to 9 bits, low digit first: a histogram and
// a scatter launch per digit), then the sorted list is cut into pieces of
// kPiece pairs that are summed independently, so a token's share of the work
// does not depend on how often it occurs.  A run of one token that crosses a
// piece border leaves float32 partial sums, which a last launch adds in order.
// Tokens that are padding or out of range get the key `vocab` and sort last.
// ---------------------------------------------------------------------------
constexpr int kRadixBits = 9;
constexpr int kRadix = 1 << kRadixBits;
constexpr int kSortThreads = 256;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortItems = 8;
constexpr int kSortTile = kSortThreads * kSortItems;   // keys of a CTA's inner step
constexpr int kSortMaxTiles = 512;                     // rows of the histogram table
constexpr int kPiece = 64;

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
  int* counter;               // crossing runs found later; reset in the first pass
  int* err;
};

// hist[tile][digit] of one pass.
__global__ void __launch_bounds__(kSortThreads) sort_hist_kernel(SortPass p) {
  __shared__ uint32_t h[kRadix];
  for (int i = threadIdx.x; i < kRadix; i += kSortThreads) h[i] = 0;
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
  __shared__ uint32_t base[kRadix];                 // next output slot of each digit
  __shared__ uint32_t cnt[kSortWarps][kRadix];
  __shared__ uint32_t wsum[kSortWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int C = kRadix / kSortThreads;          // digits per thread (consecutive)
  uint32_t tot[C], before[C], run = 0;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int d = threadIdx.x * C + c;
    uint32_t t = 0, b = 0;
#pragma unroll 4
    for (int k = 0; k < (int)gridDim.x; ++k) {
      const uint32_t h = p.hist[(int64_t)k * kRadix + d];
      t += h;
      if (k < (int)blockIdx.x) b += h;
    }
    tot[c] = t;
    before[c] = b;
    run += t;
  }
  uint32_t incl = run;                              // inclusive scan over threads
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) wsum[warp] = incl;
  __syncthreads();
  uint32_t off = incl - run;
  for (int w = 0; w < warp; ++w) off += wsum[w];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    base[threadIdx.x * C + c] = off + before[c];
    off += tot[c];
  }
  const uint32_t mask = (1u << p.bits) - 1;
  const int64_t lo = (int64_t)blockIdx.x * p.tile;
  const int64_t hi = lo + p.tile < p.n ? lo + p.tile : p.n;
  for (int64_t t0 = lo; t0 < hi; t0 += kSortTile) {
    __syncthreads();
    for (int i = threadIdx.x; i < kSortWarps * kRadix; i += kSortThreads) (&cnt[0][0])[i] = 0;
    __syncthreads();
    uint32_t key[kSortItems], row[kSortItems], rank[kSortItems];
#pragma unroll
    for (int r = 0; r < kSortItems; ++r) {
      const int64_t i = t0 + warp * (32 * kSortItems) + r * 32 + lane;
      const bool in = i < hi;
      if (in) {
        key[r] = p.keys ? p.keys[i] : token_key(p.ids, i, p.vocab, p.pad, nullptr);
        row[r] = p.keys ? p.rows[i] : (uint32_t)i;
      }
      const uint32_t d = in ? (key[r] >> p.shift) & mask : kRadix;   // kRadix: no key
      const uint32_t same = __match_any_sync(0xffffffffu, d);
      const int before_me = __popc(same & ((1u << lane) - 1));
      if (in) rank[r] = cnt[warp][d] + before_me;
      __syncwarp();
      if (in && before_me == 0) cnt[warp][d] += __popc(same);
      __syncwarp();
    }
    __syncthreads();
    for (int d = threadIdx.x; d < kRadix; d += kSortThreads) {
      uint32_t o = base[d];
#pragma unroll
      for (int w = 0; w < kSortWarps; ++w) {
        const uint32_t x = cnt[w][d];
        cnt[w][d] = o;
        o += x;
      }
      base[d] = o;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kSortItems; ++r) {
      const int64_t i = t0 + warp * (32 * kSortItems) + r * 32 + lane;
      if (i < hi) {
        const uint32_t pos = cnt[warp][(key[r] >> p.shift) & mask] + rank[r];
        p.out_keys[pos] = key[r];
        p.out_rows[pos] = row[r];
      }
    }
  }
}

// First position in the sorted keys that is not below `key`.
__device__ __forceinline__ int64_t lower_bound(const uint32_t* __restrict__ keys, int64_t n,
                                               uint32_t key) {
  int64_t lo = 0, hi = n;
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (__ldg(keys + mid) < key) lo = mid + 1; else hi = mid;
  }
  return lo;
}

struct GradParams {
  int64_t n, vocab;
  uint32_t vpr;               // 16-byte vectors per row
  const uint32_t* keys;       // sorted
  const uint32_t* rows;
  float scale;
  float* part;                // [pieces][2][dim]: head / tail sums of crossing runs
  int* counter;               // number of crossing runs
  uint32_t* owners;           // the piece each crossing run starts in
  int64_t pieces;
  int zero_blocks;            // leading CTAs (x) that clear rows of absent tokens
};

constexpr int kZeroRows = 32;   // rows of dW per clearing CTA
constexpr int kGradUnroll = 8;  // rows in flight per thread

// grid.x: zero_blocks clearing CTAs, then one CTA per piece; grid.y: 128
// vectors of the width each.
template <typename T>
__global__ void __launch_bounds__(kGradThreads)
grad_pieces_kernel(GradParams p, const T* __restrict__ dy, T* __restrict__ dw) {
  using V = Vec<T>;
  constexpr int E = V::kElems;
  __shared__ uint32_t skey[kPiece + 2];   // keys of the piece and its neighbours
  __shared__ uint32_t srow[kPiece];
  const uint32_t vec = blockIdx.y * kGradThreads + threadIdx.x;
  const bool active = vec < p.vpr;
  if ((int)blockIdx.x < p.zero_blocks) {
    const int64_t v0 = (int64_t)blockIdx.x * kZeroRows;
    if (threadIdx.x < kZeroRows) {
      const int64_t v = v0 + threadIdx.x;
      uint32_t absent = 0;
      if (v < p.vocab) {
        const int64_t at = lower_bound(p.keys, p.n, (uint32_t)v);
        absent = at == p.n || p.keys[at] != (uint32_t)v;
      }
      srow[threadIdx.x] = absent;
    }
    __syncthreads();
    if (active)
      for (int r = 0; r < kZeroRows; ++r)
        if (srow[r]) stg16(dw + ((v0 + r) * p.vpr + vec) * E, make_uint4(0, 0, 0, 0));
    return;
  }
  const int64_t piece = blockIdx.x - p.zero_blocks;
  const int64_t first = piece * kPiece;
  const uint32_t none = 0xffffffffu;
  for (int i = threadIdx.x; i < kPiece + 2; i += kGradThreads) {
    const int64_t at = first + i - 1;
    skey[i] = at >= 0 && at < p.n ? __ldg(p.keys + at) : none;
    if (i >= 1 && i <= kPiece && at < p.n) srow[i - 1] = __ldg(p.rows + at);
  }
  __syncthreads();
  // entries of the piece: up to the end of the list or the dropped tokens
  int len = p.n - first < kPiece ? (int)(p.n - first) : kPiece;
  while (len > 0 && skey[len] >= (uint32_t)p.vocab) --len;
  if (len == 0) return;
  if (blockIdx.y == 0 && threadIdx.x == 0 && len == kPiece && skey[kPiece] == skey[kPiece + 1]) {
    // the last run crosses into the next piece; listed where it starts (keys
    // ascend: if the entry before the piece has its key, all of the piece does)
    const bool starts = skey[0] != skey[kPiece];
    if (starts) p.owners[atomicAdd(p.counter, 1)] = (uint32_t)piece;
  }
  if (!active) return;
  const int64_t dim = (int64_t)p.vpr * E;
  bool head = skey[0] == skey[1];         // the first run began in an earlier piece
  float acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  for (int j0 = 0; j0 < len; j0 += kGradUnroll) {
    uint4 x[kGradUnroll];
#pragma unroll
    for (int u = 0; u < kGradUnroll; ++u)
      if (j0 + u < len) x[u] = ldg16_stream(dy + ((int64_t)srow[j0 + u] * p.vpr + vec) * E);
#pragma unroll
    for (int u = 0; u < kGradUnroll; ++u) {
      const int j = j0 + u;
      if (j < len) {
        float f[E];
        V::to_float(x[u], f);
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] += f[e];
        const uint32_t key = skey[j + 1];
        const bool more = skey[j + 2] == key;
        if (!more || j + 1 == len) {
          if (head || more) {
            float* dst = p.part + (piece * 2 + (head ? 0 : 1)) * dim + (int64_t)vec * E;
#pragma unroll
            for (int e = 0; e < E; e += 4)
              *reinterpret_cast<float4*>(dst + e) =
                  make_float4(acc[e], acc[e + 1], acc[e + 2], acc[e + 3]);
          } else {
            store_scaled<T>(dw + ((int64_t)key * p.vpr + vec) * E, acc, p.scale);
          }
          head = false;
#pragma unroll
          for (int e = 0; e < E; ++e) acc[e] = 0.f;
        }
      }
    }
  }
}

// Joins the partial sums of the runs that cross pieces.  A task is (run, 128
// columns); its warps take every kJoinWarps-th partial, then add up in order.
constexpr int kJoinWarps = 8;

template <typename T>
__global__ void __launch_bounds__(kJoinWarps * 32)
grad_join_kernel(GradParams p, T* __restrict__ dw) {
  __shared__ float4 sum[kJoinWarps][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t dim = (int64_t)p.vpr * Vec<T>::kElems;
  const int64_t chunks = (dim + 127) / 128;
  const int64_t tasks = (int64_t)*p.counter * chunks;
  for (int64_t t = blockIdx.x; t < tasks; t += gridDim.x) {
    const int64_t piece = p.owners[t / chunks];
    const int64_t col = (t % chunks) * 128 + lane * 4;
    const uint32_t key = p.keys[piece * kPiece + kPiece - 1];
    const int64_t last = (lower_bound(p.keys, p.n, key + 1) - 1) / kPiece;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    if (col < dim) {
      for (int64_t q = piece + warp; q <= last; q += kJoinWarps) {
        const float4 x = *reinterpret_cast<const float4*>(
            p.part + (q * 2 + (q == piece ? 1 : 0)) * dim + col);
        a.x += x.x; a.y += x.y; a.z += x.z; a.w += x.w;
      }
    }
    sum[warp][lane] = a;
    __syncthreads();
    if (warp == 0 && col < dim) {
      for (int w = 1; w < kJoinWarps; ++w) {
        const float4 x = sum[w][lane];
        a.x += x.x; a.y += x.y; a.z += x.z; a.w += x.w;
      }
      T* dst = dw + (int64_t)key * dim + col;
      dst[0] = from_f32<T>(a.x * p.scale);
      dst[1] = from_f32<T>(a.y * p.scale);
      dst[2] = from_f32<T>(a.z * p.scale);
      dst[3] = from_f32<T>(a.w * p.scale);
    }
    __syncthreads();
  }
}

}  // namespace embed
}  // namespace esa
