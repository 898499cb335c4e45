// Log probabilities of given tokens, with the entropy and the top alternatives
// of each row of logits, and their gradient.
//
// Forward, one pass over a row x[0..V) (z = x - m, m the row's maximum):
//   S0 = sum e^z, S1 = sum e^z z      (float32, rescaled when m grows)
//   log p_t = z_t - ln S0,   H = -sum p ln p = ln S0 - S1 / S0
// m is subtracted before the product with log2(e), so logits of any magnitude
// (a mask of the type's lowest value included) keep their differences.  A row
// with a NaN or +infinity gives NaN, so does a row of -infinity alone.
//
// Backward: dx_j = g ([j = t] - p_j) - h p_j (ln p_j + H).
//
// Top alternatives: order by value (NaN above all), then by the lower index; as
// one 64-bit key per element no two are equal.  The pass leaves each thread with
// the maximum of its own elements.  The k-th largest of the maxima of at least 2 k
// groups of threads is a lower bound of the k-th largest element, so only the
// threads at or above it hold candidates: their warps read those few threads'
// elements again (from L1 / L2) and keep a sorted list of 32, one key per lane.
// The lists of the warps, then of the CTAs of a row, are merged two by two.
//
// A row belongs to a cluster of 1, 2, 4 or 8 CTAs (few rows: more CTAs per row),
// joined through distributed shared memory in the same launch.
//
// What bounds it: the forward pass makes an exponential per element.  8192 x 32000 bf16
// takes 84 us (95 % of the measured copy rate), 105 with five alternatives; the
// special-function pipe is busy for three quarters of it, and some 7.5 instructions per
// element, few by packed maxima, mixed-precision differences and packed float32 sums,
// fill 64 % of the issue slots.  The gradient takes 176 us (91 %).  8 rows of 32000, 20
// alternatives: 6.5 us, 3.4 without: a chain of short sorts.  With fewer finite groups
// than alternatives the bound is -infinity and every element is looked at again: with
// 10 tokens left of those 32000 it takes 35 us.
#pragma once
#include <cooperative_groups.h>

#include "esa_f32x2.cuh"

namespace esa {
namespace score {

constexpr int kErrToken = 16;      // ESA_DEVERR_TOKEN_RANGE
constexpr int kMaxTop = 32;        // one list entry per lane
constexpr int64_t kIgnore = -100;  // token of a row without a log probability
constexpr float kLowest = -3.4028234663852886e38f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kUnroll = 4;         // vectors in flight per thread

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Unsigned order of float32 values: NaN highest, -0 equal to +0.
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t o) {
  return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);   // 0xffffffff: a NaN
}
__device__ __forceinline__ uint64_t key_of(float x, uint32_t idx) {
  return (uint64_t)order_of(x) << 32 | (uint32_t)~idx;
}

// Lists of 32 in descending order, one entry per lane.
template <typename K> __device__ __forceinline__ K pick(K a, K b, bool larger) {
  return (a > b) == larger ? a : b;
}
// A sequence that rises and falls once -> descending.
template <typename K> __device__ __forceinline__ K settle(K v, int lane) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    v = pick(v, __shfl_xor_sync(0xffffffffu, v, o), (lane & o) == 0);
  return v;
}
template <typename K> __device__ __forceinline__ K sort32(K v, int lane) {
#pragma unroll
  for (int n = 2; n <= 32; n <<= 1)
#pragma unroll
    for (int o = n / 2; o > 0; o >>= 1)
      v = pick(v, __shfl_xor_sync(0xffffffffu, v, o), ((lane & o) == 0) == ((lane & n) == 0 || n == 32));
  return v;
}
// The 32 largest of two descending lists; `other` is read in reverse by lane.
template <typename K> __device__ __forceinline__ K merge32(K mine, K other_reversed, int lane) {
  return settle(mine > other_reversed ? mine : other_reversed, lane);
}

struct Stats { float m, s0, s1; };

// Largest of the warp's values, none a NaN: their bits in the order of signed integers.
__device__ __forceinline__ float max_of_warp(float x) {
  const int b = __float_as_int(x);
  const int m = __reduce_max_sync(0xffffffffu, b ^ ((b >> 31) & 0x7fffffff));
  return __int_as_float(m ^ ((m >> 31) & 0x7fffffff));
}

// The step of m when it grows; its exponential is 0 long before the bound, which
// keeps its product with a sum finite.
__device__ __forceinline__ float rescale(float from, float to) { return fmaxf(from - to, -1e25f); }

__device__ __forceinline__ Stats join(const Stats& a, const Stats& b) {
  Stats r;
  r.m = fmaxf(a.m, b.m);
  const float da = rescale(a.m, r.m), db = rescale(b.m, r.m);
  const float ea = ex2(da * kLog2e), eb = ex2(db * kLog2e);
  r.s0 = a.s0 * ea + b.s0 * eb;
  r.s1 = ea * (a.s1 + da * a.s0) + eb * (b.s1 + db * b.s0);
  return r;
}

// Two 16-bit elements: the larger ones (NaNs passed over, or kept), x - m in float32.
template <typename T> struct Pair;
// kFloor: elements below it count as it, which keeps -infinity out of the products;
// next to a maximum of kSafe or more their exponential is 0 either way.  No difference
// from a maximum of the type may reach -infinity: -2^100 less bfloat16's largest value,
// (2 - 2^-7) 2^127, is within float32, -2^126 less it would not be.
#define ESA_PAIR(T, PTXTYPE, ONE, FLOOR2, NONE, FLOOR, SAFE)                                 \
  template <> struct Pair<T> {                                                               \
    static constexpr uint32_t kFloor2 = FLOOR2, kNone = NONE;                                \
    static constexpr float kFloor = FLOOR, kSafe = SAFE;                                     \
    __device__ __forceinline__ static uint32_t larger(uint32_t a, uint32_t b) {              \
      uint32_t r;                                                                            \
      asm("max." PTXTYPE "x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));                       \
      return r;                                                                              \
    }                                                                                        \
    __device__ __forceinline__ static uint32_t larger_nan(uint32_t a, uint32_t b) {          \
      uint32_t r;                                                                            \
      asm("max.NaN." PTXTYPE "x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));                   \
      return r;                                                                              \
    }                                                                                        \
    /* the products with one are exact: two conversions and two sums in two instructions */  \
    __device__ __forceinline__ static void minus(uint32_t x, float neg_m, float& a, float& b) { \
      asm("{\n\t.reg .b16 l, h, one;\n\tmov.b32 {l, h}, %2;\n\tmov.b16 one, " ONE ";\n\t"     \
          "fma.rn.f32." PTXTYPE " %0, l, one, %3;\n\tfma.rn.f32." PTXTYPE " %1, h, one, %3;\n\t}" \
          : "=f"(a), "=f"(b)                                                                 \
          : "r"(x), "f"(neg_m));                                                             \
    }                                                                                        \
  };
ESA_PAIR(__nv_bfloat16, "bf16", "0x3F80", 0xf180f180u, 0xff80ff80u, -0x1p100f, -0x1p99f)
ESA_PAIR(__half, "f16", "0x3C00", 0xfbfffbffu, 0xfc00fc00u, -65504.f, -65000.f)
#undef ESA_PAIR
template <> struct Pair<float> {
  static constexpr uint32_t kNone = 0xff800000u;
  static constexpr float kFloor = kLowest, kSafe = -INFINITY;      // nothing is raised
};

__device__ __forceinline__ uint32_t word_of(const uint4& v, int i) {
  return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}

// Largest of the elements of the vectors; NaNs are passed over.
template <typename T> __device__ __forceinline__ float vec_max(const uint4 (&x)[kUnroll]) {
  if constexpr (std::is_same<T, float>::value) {
    float m = -INFINITY;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      m = fmaxf(fmaxf(fmaxf(m, __uint_as_float(x[u].x)), fmaxf(__uint_as_float(x[u].y), __uint_as_float(x[u].z))),
                __uint_as_float(x[u].w));
    return m;
  } else {
    uint32_t m = Pair<T>::kNone;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) m = Pair<T>::larger(m, word_of(x[u], i));
    float a, b;
    Pair<T>::minus(m, -0.f, a, b);
    return fmaxf(a, b);
  }
}

__device__ __forceinline__ void grow(Stats& s, float m) {
  if (m > s.m) {
    const float d = rescale(s.m, m), e = ex2(d * kLog2e);
    s.s1 = e * (s.s1 + d * s.s0);
    s.s0 *= e;
    s.m = m;
  }
}

// One element more (the ragged ends of a row).
__device__ __forceinline__ void add_one(Stats& s, float x) {
  grow(s, fmaxf(x, kLowest));
  const float z = x - s.m, e = ex2(z * kLog2e);
  s.s0 += e;
  s.s1 = fmaf(e, fmaxf(z, kLowest), s.s1);
}

// The elements of a row that whole 16-byte vectors cover, and those before and after.
template <typename T> struct RowParts {
  const uint4* body;
  int head, tail;        // single elements before / after the body
  int64_t nvec;
  __device__ __forceinline__ RowParts(const T* row, int64_t V) {
    constexpr int E = Vec<T>::kElems;
    const int to_border = (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / (int)sizeof(T);
    head = (int)(to_border < V ? to_border : V);
    nvec = (V - head) / E;
    tail = (int)(V - head - nvec * E);
    body = reinterpret_cast<const uint4*>(row + head);
  }
};

template <typename T> struct FwdParams {
  const T* logits;
  int64_t stride, V;
  const void* tokens;
  int id_bytes, top;
  float *logprobs, *entropy;
  float2* stats;          // (m, ln S0)
  int64_t* top_ids;
  float* top_logprobs;
  int* err;
};

__device__ __forceinline__ int64_t load_token(const void* tokens, int id_bytes, int64_t row) {
  return id_bytes == 8 ? static_cast<const int64_t*>(tokens)[row]
                       : (int64_t)static_cast<const int32_t*>(tokens)[row];
}

template <typename T, int NW, bool TOP>
__global__ void __launch_bounds__(NW * 32)
fwd_kernel(const FwdParams<T> p) {
  namespace cg = cooperative_groups;
  constexpr int E = Vec<T>::kElems;
  __shared__ __align__(16) Stats s_stats[NW];
  __shared__ Stats s_cta;                       // read by the other CTAs of the row
  __shared__ float s_max[64];
  __shared__ float s_bound;
  __shared__ int s_count;
  __shared__ uint64_t s_list[TOP ? NW : 1][32];  // also the elements found
  cudaGridDependencySynchronize();
  const cg::cluster_group cluster = cg::this_cluster();
  const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = blockIdx.x / ctas;
  const T* x = p.logits + row * p.stride;
  const RowParts<T> parts(x, p.V);
  const int nvec = (int)parts.nvec;                  // < 2^29
  const int step = ctas * NW * 32, first = rank * NW * 32 + threadIdx.x;

  Stats s = {Pair<T>::kFloor, 0.f, 0.f};
  float own_max = -INFINITY;
  for (int i = first; i < nvec; i += kUnroll * step) {
    uint4 v[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const uint32_t none = Pair<T>::kNone;
      v[u] = make_uint4(none, none, none, none);
      if (i + u * step < nvec) v[u] = ld16(parts.body + i + u * step);
    }
    own_max = fmaxf(own_max, vec_max<T>(v));
    grow(s, own_max);
    F2 s0 = f2(0.f, 0.f), s1 = f2(0.f, 0.f);
    const F2 l2e = f2(kLog2e, kLog2e);
    auto add = [&](float za, float zb) {
      float a, b;
      split(mul2(f2(za, zb), l2e), a, b);
      const F2 pe = f2(ex2(a), ex2(b));
      s0 = add2(s0, pe);
      return pe;
    };
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
      for (int e = 0; e < 4; e += sizeof(T) == 4 ? 2 : 1) {
        float za, zb;
        if constexpr (sizeof(T) == 4) {
          za = __uint_as_float(word_of(v[u], e)) - s.m;
          zb = __uint_as_float(word_of(v[u], e + 1)) - s.m;
          const F2 pe = add(za, zb);
          s1 = fma2(pe, f2(fmaxf(za, kLowest), fmaxf(zb, kLowest)), s1);   // 0 * -inf is 0 here
        } else {
          Pair<T>::minus(Pair<T>::larger_nan(word_of(v[u], e), Pair<T>::kFloor2), -s.m, za, zb);
          s1 = fma2(add(za, zb), f2(za, zb), s1);
        }
      }
    float a, b;
    split(s0, a, b);
    s.s0 += a + b;
    split(s1, a, b);
    s.s1 += a + b;
  }
  const float warp_max = max_of_warp(own_max);
  if (warp_max == -INFINITY) {         // nothing, or -infinity (and NaNs) alone
    if (s.s0 == s.s0) s = {kLowest, 0.f, 0.f};
  } else if (warp_max < Pair<T>::kSafe) {
    // what was raised to the floor does count here: element by element
    s = {kLowest, 0.f, 0.f};
    for (int i = first; i < nvec; i += step)
      for (int e = 0; e < E; ++e) add_one(s, (float)x[parts.head + (int64_t)i * E + e]);
  }
  // the ragged ends: at most 2 (E - 1) < 32 elements, one per lane of one warp
  int64_t edge = -1;
  if (rank == 0 && warp == 0) {
    if (lane < parts.head) edge = lane;
    else if (lane < parts.head + parts.tail) edge = (int64_t)nvec * E + lane;
    if (edge >= 0) add_one(s, (float)x[edge]);
  }
  {
    const float m = max_of_warp(s.m), d = rescale(s.m, m), e = ex2(d * kLog2e), s0 = s.s0;
    s = {m, warp_sum(s0 * e), warp_sum(e * (s.s1 + d * s0))};
  }
  if (lane == 0) s_stats[warp] = s;
  bool nans = false;
  float bound = -INFINITY;
  if constexpr (TOP) {
    // maxima of groups of `span` lanes, at least 2 k of them where there are as many
    int span = 32;
    while (span > 1 && NW * 32 / span < 2 * p.top) span >>= 1;
    float gm = own_max;
    for (int o = span >> 1; o > 0; o >>= 1) gm = fmaxf(gm, __shfl_xor_sync(0xffffffffu, gm, o));
    if (threadIdx.x < 64) s_max[threadIdx.x] = -INFINITY;
    __syncthreads();
    if (lane % span == 0) s_max[threadIdx.x / span] = gm;
    nans = __syncthreads_or(s.s0 != s.s0);
    if (warp == 0) {
      float top = sort32(s_max[lane], lane);
      if (NW * 32 / span > 32) {
        const float b = sort32(s_max[32 + lane], lane);
        top = merge32(top, __shfl_xor_sync(0xffffffffu, b, 31), lane);
      }
      if (lane == p.top - 1) s_bound = top;
      if (lane == 0) s_count = 0;
    }
  }
  __syncthreads();

  uint64_t list = 0;           // below every real key
  if constexpr (TOP) {
    // NaNs are above every bound, and what is masked below those there are
    const bool all = nans || s_bound == -INFINITY;
    if (!all) bound = s_bound;
    // Few elements reach the bound as a rule: a list of all of them, sorted by one
    // warp (whose order does not depend on that of the list).
    constexpr int kMost = 64;
    uint64_t* const found = &s_list[0][0];
    bool listed = !all;
    if (listed) {
      auto add = [&](float v, int64_t idx) {
        const int at = atomicAdd(&s_count, 1);
        if (at < kMost) found[at] = key_of(v, (uint32_t)idx);
      };
      if (edge >= 0 && (float)x[edge] >= bound) add((float)x[edge], edge);
      auto look = [&](int64_t i) {
        const uint4 v = ld16(parts.body + i);
        float f[E];
        Vec<T>::to_float(v, f);
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (f[e] >= bound) add(f[e], parts.head + i * E + e);
      };
      if (nvec <= 4 * step) {
        // few vectors each: every owner looks through its own
        if (own_max >= bound)
          for (int64_t i = first; i < nvec; i += step) look(i);
      } else {
        uint32_t owners = __ballot_sync(0xffffffffu, own_max >= bound);
        while (owners) {
          const int o = __ffs(owners) - 1;
          owners &= owners - 1;
          for (int64_t i = rank * NW * 32 + warp * 32 + o + lane * (int64_t)step; i < nvec;
               i += 32 * (int64_t)step)
            look(i);
        }
      }
      __syncthreads();
      listed = s_count <= kMost;
    }
    if (listed) {
      if (warp == 0) {
        list = sort32(lane < s_count ? found[lane] : 0, lane);
        if (s_count > 32) {
          const uint64_t b = sort32(lane + 32 < s_count ? found[lane + 32] : 0, lane);
          list = merge32(list, __shfl_xor_sync(0xffffffffu, b, 31), lane);
        }
        __syncwarp();
        s_list[0][lane] = list;
      }
    } else {
      // Many (equal values, or NaNs): each warp keeps the 32 largest of its elements.
      __syncthreads();
      uint64_t worst = 0;
      auto offer = [&](bool candidate, float v, int64_t idx) {
        const uint64_t key = candidate ? key_of(v, (uint32_t)idx) : 0;
        uint32_t mask = __ballot_sync(0xffffffffu, key > worst);
        while (mask) {
          const uint64_t c = __shfl_sync(0xffffffffu, key, __ffs(mask) - 1);
          mask &= mask - 1;
          const int at = __popc(__ballot_sync(0xffffffffu, list > c));
          const uint64_t up = __shfl_up_sync(0xffffffffu, list, 1);
          if (at < 32) list = lane < at ? list : lane == at ? c : up;
          worst = __shfl_sync(0xffffffffu, list, 31);
        }
      };
      if (rank == 0 && warp == 0) offer(edge >= 0, edge >= 0 ? (float)x[edge] : 0.f, edge);
      uint32_t owners = __ballot_sync(0xffffffffu, all || own_max >= bound);
      while (owners) {
        const int o = __ffs(owners) - 1;
        owners &= owners - 1;
        for (int64_t j = rank * NW * 32 + warp * 32 + o; j < nvec; j += 32 * (int64_t)step) {   // the same on every lane
          const int64_t i = j + lane * (int64_t)step;
          const bool in = i < nvec;
          uint4 v = make_uint4(0, 0, 0, 0);
          if (in) v = ld16(parts.body + i);
          float f[E];
          Vec<T>::to_float(v, f);
          bool some = all;
#pragma unroll
          for (int e = 0; e < E; ++e) some = some || f[e] >= bound;
          if (!__any_sync(0xffffffffu, in && some)) continue;
#pragma unroll
          for (int e = 0; e < E; ++e)
            offer(in && (all || f[e] >= bound), f[e], parts.head + i * E + e);
        }
      }
      s_list[warp][lane] = list;
      __syncthreads();
#pragma unroll
      for (int n = NW / 2; n >= 1; n >>= 1) {
        if (warp < n)
          s_list[warp][lane] = merge32(s_list[warp][lane], s_list[warp + n][31 - lane], lane);
        __syncthreads();
      }
    }
  }
  if (warp == 0) {
    s = s_stats[lane < NW ? lane : 0];
#pragma unroll
    for (int o = NW / 2; o > 0; o >>= 1) {
      Stats t;
      t.m = __shfl_xor_sync(0xffffffffu, s.m, o);
      t.s0 = __shfl_xor_sync(0xffffffffu, s.s0, o);
      t.s1 = __shfl_xor_sync(0xffffffffu, s.s1, o);
      s = join(s, t);
    }
    s.m = __shfl_sync(0xffffffffu, s.m, 0);
    s.s0 = __shfl_sync(0xffffffffu, s.s0, 0);
    s.s1 = __shfl_sync(0xffffffffu, s.s1, 0);
  }
  if (ctas > 1) {
    if (threadIdx.x == 0) s_cta = s;
    cluster.sync();
    if (rank == 0) {
      if constexpr (TOP && NW >= 8) {
        // a warp fetches the list of each CTA; they are merged two by two
        if (warp > 0 && warp < ctas) s_list[warp][lane] = *cluster.map_shared_rank(&s_list[0][lane], warp);
        __syncthreads();
        for (int n = ctas / 2; n >= 1; n >>= 1) {
          if (warp < n)
            s_list[warp][lane] = merge32(s_list[warp][lane], s_list[warp + n][31 - lane], lane);
          __syncthreads();
        }
      }
      if (warp == 0) {
        if constexpr (TOP) {
          list = s_list[0][lane];
          if constexpr (NW < 8)
            for (int r = 1; r < ctas; ++r)
              list = merge32(list, *cluster.map_shared_rank(&s_list[0][31 - lane], r), lane);
        }
        s = *cluster.map_shared_rank(&s_cta, lane & (ctas - 1));
        for (int o = ctas / 2; o > 0; o >>= 1) {
          Stats t;
          t.m = __shfl_xor_sync(0xffffffffu, s.m, o);
          t.s0 = __shfl_xor_sync(0xffffffffu, s.s0, o);
          t.s1 = __shfl_xor_sync(0xffffffffu, s.s1, o);
          s = join(s, t);
        }
        s.m = __shfl_sync(0xffffffffu, s.m, 0);
        s.s0 = __shfl_sync(0xffffffffu, s.s0, 0);
        s.s1 = __shfl_sync(0xffffffffu, s.s1, 0);
      }
    }
    cluster.sync();        // the other CTAs' shared memory lives until it is read
  } else if constexpr (TOP) {
    if (warp == 0) list = s_list[0][lane];
  }
  if (rank != 0 || warp != 0) return;
  const float log_s = logf(s.s0);
  if constexpr (TOP) {
    if (lane < p.top) {
      p.top_ids[row * p.top + lane] = (int64_t)(uint32_t)~(uint32_t)list;
      p.top_logprobs[row * p.top + lane] = value_of((uint32_t)(list >> 32)) - s.m - log_s;
    }
  }
  if (lane == 0) {
    const int64_t t = load_token(p.tokens, p.id_bytes, row);
    float lp = 0.f;
    if (t >= 0 && t < p.V) {
      lp = (float)x[t] - s.m - log_s;
    } else if (t != kIgnore) {
      lp = __uint_as_float(0x7fffffffu);
      if (p.err) atomicOr(p.err, kErrToken);
    }
    p.logprobs[row] = lp;
    p.entropy[row] = log_s - s.s1 / s.s0;
    p.stats[row] = make_float2(s.m, log_s);
  }
}

// ---------------------------------------------------------------------------
// Gradient: element by element, a CTA per kBwdVecs vectors of a row.  A row with
// neither gradient (an ignored token, no entropy gradient) is cleared unread.
// ---------------------------------------------------------------------------
constexpr int kBwdThreads = 256;
constexpr int kBwdVecs = kBwdThreads * kUnroll;

template <typename T> struct BwdParams {
  const T* logits;
  T* dlogits;
  int64_t stride, dstride, V;
  const void* tokens;
  int id_bytes;
  unsigned parts;         // CTAs per row
  const float2* stats;
  const float* entropy;
  const float* dlogprobs; // may be null: zeros
  const float* dentropy;  // may be null: zeros
  int* err;
};

struct RowGrad {
  float m, shift, a, h, g;    // p = 2^(log2e (x - m) - shift); dx = -p (a + h (x - m))
  __device__ __forceinline__ float operator()(float x) const {
    const float z = x - m;
    const float pr = ex2(fmaf(z, kLog2e, -shift));
    // p is 0 below z = -1e4, the product with an infinite z is not
    return -pr * fmaf(h, fmaxf(z, -1e4f), a);
  }
};

template <typename T>
__global__ void __launch_bounds__(kBwdThreads)
bwd_kernel(const BwdParams<T> p) {
  constexpr int E = Vec<T>::kElems;
  const int64_t row = blockIdx.x / p.parts;
  const unsigned part = blockIdx.x % p.parts;
  const T* x = p.logits + row * p.stride;
  T* dx = p.dlogits + row * p.dstride;
  const RowParts<T> parts(x, p.V);
  int64_t t = load_token(p.tokens, p.id_bytes, row);
  RowGrad r;
  r.g = p.dlogprobs && t != kIgnore ? p.dlogprobs[row] : 0.f;
  r.h = p.dentropy ? p.dentropy[row] : 0.f;
  const bool none = r.g == 0.f && r.h == 0.f;
  const float2 st = p.stats[row];
  r.m = st.x;
  r.shift = st.y * kLog2e;
  // g + h (ln p + H) with ln p = x - m - ln S0
  r.a = r.h == 0.f ? r.g : fmaf(r.h, p.entropy[row] - st.y, r.g);
  if (t != kIgnore && (t < 0 || t >= p.V)) {
    if (r.g != 0.f) r.a = __uint_as_float(0x7fffffffu);     // as the forward's NaN
    if (p.err && part == 0 && threadIdx.x == 0) atomicOr(p.err, kErrToken);
  }
  if (t < 0 || t >= p.V) t = -1;
  auto one = [&](int64_t j) {
    float d = none ? 0.f : r((float)x[j]);
    if (j == t) d += r.g;
    dx[j] = from_f32<T>(d);
  };
  if (part == 0 && threadIdx.x < 32) {
    const int lane = threadIdx.x;
    if (lane < parts.head) one(lane);
    else if (lane < parts.head + parts.tail) one(parts.nvec * E + lane);
  }
  const int64_t base = (int64_t)part * kBwdVecs + threadIdx.x;
  uint4 v[kUnroll];
  if (!none) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t i = base + u * kBwdThreads;
      if (i < parts.nvec) v[u] = parts.body[i];   // dlogits may be logits: no read-only load
    }
  }
  // vectors of logits and gradient start at the same elements (equal strides)?
  const bool same = ((reinterpret_cast<uintptr_t>(dx + parts.head)) & 15) == 0;
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int64_t i = base + u * kBwdThreads;
    if (i >= parts.nvec) break;
    const int64_t j0 = parts.head + i * E;
    float f[E];
    if (none) {
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] = 0.f;
    } else {
      Vec<T>::to_float(v[u], f);
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] = r(f[e]);
      if (t >= j0 && t < j0 + E) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (t == j0 + e) f[e] += r.g;
      }
    }
    if (same) {
      stg16(dx + j0, Vec<T>::from_float(f));
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) dx[j0 + e] = from_f32<T>(f[e]);
    }
  }
}

}  // namespace score
}  // namespace esa
