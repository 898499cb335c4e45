// Per-head RMS normalisation of queries and keys with the rotary embedding in
// the same pass.  For a head row x of D elements at position p, i < D/2:
//
//   rstd = (mean(x^2) + eps)^(-1/2),   n = x * rstd * w
//   out[i]       = n[i] cos a - n[i + D/2] sin a
//   out[i + D/2] = n[i + D/2] cos a + n[i] sin a,      a = p * inv_freq[i]
//
// and the backward, with dn the inverse rotation of dout, xh = x * rstd:
//
//   dx = rstd * (w dn - xh mean(xh w dn)),   dw = sum over rows of dn xh
//
// A row is held by D / (2 E) threads: thread t owns elements [tE, tE + E) and
// the same of the second half, so the rotation needs no exchange.  The forward
// has E = one 16-byte vector.  The backward, which holds twice the operands
// and the weight gradient's sums, has E = 4, so that several rounds fit in the
// registers.  A warp takes the heads of one token, 32 / threads-per-row
// at a time (a round), and loads kUnroll rounds before it works on the first:
// the kernels are HBM-bound (every element is read and written once) and need
// that many bytes in flight.  The D / 2 angles of a token are formed once,
// spread over the warp's lanes, and shared through shared memory.  rstd is
// formed again in the backward instead of being kept.
//
// Where the heads of a token do not fill a warp's rounds, a task is several
// tokens, whose rows (token by token, head by head) the rounds run through.
#pragma once
#include "esa_f32x2.cuh"

namespace esa {
namespace qknorm {

template <typename T>
struct Heads {          // the query or the key side of a call
  const T* x; int64_t xb, xh, xs;
  const T* d; int64_t db, dh, ds;     // gradient of the output (backward)
  T* o; int64_t ob, oh, os;           // output, or gradient of x
  const T* w;
  int H;
};

template <typename T>
struct Params {
  Heads<T> q, k;
  int64_t L, tokens;                  // positions per batch entry, B * L
  const int64_t* pos;                 // nullptr: 0 .. L-1
  int64_t pos_sb;                     // 0: positions shared by the batch
  const float* inv_freq;
  float eps;
  int rq, rk;                         // rounds of the query / key heads
  int rpt, tasks;                     // forward: rounds per warp task, tasks per token
  int rpt_q, rpt_k, tasks_q, tasks_k; // backward: the same for each side
  int nt, nt_q, nt_k;                 // few heads: tokens per warp task (> 1)
};

// cos and sin of p * f: the product in float64 (p and f are exact there), in
// turns, so that far positions lose nothing to the reduction.  What is left is
// at most half a turn: 16-bit types take the hardware's sine and cosine of it
// (absolute error 2^-21 on [-pi, pi], against half steps of 2^-9 and 2^-12 of
// the results), float32 the library's.
template <typename T>
__device__ __forceinline__ void rotation(int64_t p, float f, float& c, float& s) {
  double t = (double)p * (double)f * 0.15915494309189533577;   // 1 / (2 pi)
  t -= rint(t);
  if constexpr (sizeof(T) == 4) {
    sincospif((float)(2.0 * t), &s, &c);
  } else {
    const float a = (float)t * 6.2831853071795864769f;
    s = __sinf(a);
    c = __cosf(a);
  }
}

template <int TPR>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = TPR / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;

// Rounds loaded together and CTAs per SM.  Forward: two rounds on 32 warps per
// SM (65536 tokens of 40 heads of 128, bf16: 205 us; on 24 warps 222, five
// rounds on 20 warps 208).  Backward: four (two in float32), the next four
// loaded ahead, on 12 warps (32768 tokens of 64 heads: 251 us; two ahead of two
// on 16 warps 268, four without loading ahead 277).  In long runs the power
// limit lowers the SM clock and these become 213-225 and 269-283 us; a plain
// copy of as many bytes (209 us) does not reach it.
constexpr int kFwdUnroll = 2;
constexpr int kFwdCtasPerSm = 8;
template <typename T> constexpr int kBwdUnroll = sizeof(T) == 4 ? 2 : 4;
constexpr int kFewRounds = 2;         // of fwd_few_kernel: rows of at most so many rounds
constexpr int kBwdCtasPerSm = 3;

// Sums of a and b over the TPR lanes of a row, both on every lane: even lanes
// carry a through the levels, odd lanes b, so the pair costs one shuffle per
// level and one more.
template <int TPR>
__device__ __forceinline__ void row_sum2(float& a, float& b) {
  if constexpr (TPR == 1) return;
  const bool odd = threadIdx.x & 1;
  float mine = (odd ? b : a) + __shfl_xor_sync(0xffffffffu, odd ? a : b, 1);
#pragma unroll
  for (int o = 2; o < TPR; o <<= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  const float other = __shfl_xor_sync(0xffffffffu, mine, 1);
  a = odd ? other : mine;
  b = odd ? mine : other;
}

// E = 4 elements of T: 8 bytes of a 16-bit type, 16 of float32.
template <typename T> struct Quad {
  using Raw = uint2;
  __device__ __forceinline__ static void to_float(const Raw& r, F2 (&f)[2]) {
    float t[8];
    Vec<T>::to_float(make_uint4(r.x, r.y, 0, 0), t);
    f[0] = f2(t[0], t[1]);
    f[1] = f2(t[2], t[3]);
  }
  __device__ __forceinline__ static Raw from_float(const F2 (&f)[2]) {
    float t[4];
    split(f[0], t[0], t[1]);
    split(f[1], t[2], t[3]);
    return make_uint2(Vec<T>::pack(t[0], t[1]), Vec<T>::pack(t[2], t[3]));
  }
  __device__ __forceinline__ static Raw zero() { return make_uint2(0, 0); }
};
template <> struct Quad<float> {
  using Raw = uint4;
  __device__ __forceinline__ static void to_float(const Raw& r, F2 (&f)[2]) {
    f[0] = f2(__uint_as_float(r.x), __uint_as_float(r.y));
    f[1] = f2(__uint_as_float(r.z), __uint_as_float(r.w));
  }
  __device__ __forceinline__ static Raw from_float(const F2 (&f)[2]) {
    float t[4];
    split(f[0], t[0], t[1]);
    split(f[1], t[2], t[3]);
    return Vec<float>::from_float(t);
  }
  __device__ __forceinline__ static Raw zero() { return make_uint4(0, 0, 0, 0); }
};

// cos and sin of the token at `pos` for this thread's elements, by way of the
// warp's row cs_of_warp (cos of each angle, then sin).
template <typename T, int D, int E>
__device__ __forceinline__ void token_rotation(int64_t pos, const float* inv_freq, int lane, int i0,
                                               float* cs_of_warp, float (&cs)[E], float (&sn)[E]) {
  __syncwarp();      // the row's last readers are done
  for (int i = lane; i < D / 2; i += 32) {
    float c, s;
    rotation<T>(pos, inv_freq[i], c, s);
    cs_of_warp[i] = c;
    cs_of_warp[D / 2 + i] = s;
  }
  __syncwarp();
#pragma unroll
  for (int e = 0; e < E; ++e) {
    cs[e] = cs_of_warp[i0 + e];
    sn[e] = cs_of_warp[D / 2 + i0 + e];
  }
}

// The same for nt tokens from tok0 on: rows of D floats in the warp's table.
template <int D, typename T>
__device__ __forceinline__ void fill_rotations(const Params<T>& p, uint32_t tok0, int nt, int lane,
                                               float* table) {
  __syncwarp();
  for (int i = lane; i < nt * (D / 2); i += 32) {
    const int t = i / (D / 2), a = i % (D / 2);
    const uint32_t tok = tok0 + t, b = tok / (uint32_t)p.L, l = tok - b * (uint32_t)p.L;
    float c, s;
    rotation<T>(p.pos ? p.pos[b * p.pos_sb + l] : (int64_t)l, p.inv_freq[a], c, s);
    table[t * D + a] = c;
    table[t * D + D / 2 + a] = s;
  }
  __syncwarp();
}

// Pairs of a 16-byte vector.
template <typename T>
__device__ __forceinline__ void to_pairs(const uint4& raw, F2 (&f)[Vec<T>::kElems / 2]) {
  float t[Vec<T>::kElems];
  Vec<T>::to_float(raw, t);
#pragma unroll
  for (int v = 0; v < Vec<T>::kElems / 2; ++v) f[v] = f2(t[2 * v], t[2 * v + 1]);
}
template <typename T>
__device__ __forceinline__ uint4 from_pairs(const F2 (&f)[Vec<T>::kElems / 2]) {
  float t[Vec<T>::kElems];
#pragma unroll
  for (int v = 0; v < Vec<T>::kElems / 2; ++v) split(f[v], t[2 * v], t[2 * v + 1]);
  return Vec<T>::from_float(t);
}

template <typename T, int TPR>
__global__ void __launch_bounds__(kThreads, kFwdCtasPerSm) fwd_kernel(Params<T> p) {
  constexpr int E = Vec<T>::kElems;
  constexpr int P = E / 2;
  constexpr int RPW = 32 / TPR;               // rows a warp holds at once
  constexpr int D = 2 * E * TPR;
  constexpr int U = kFwdUnroll;
  __shared__ float table[kWarps][D];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // 64-bit divisions here would be an eighth of the kernel's instructions
  const uint32_t task = blockIdx.x * kWarps + warp;
  const uint32_t tok = task / (uint32_t)p.tasks;
  if (tok >= p.tokens) return;
  const uint32_t bu = tok / (uint32_t)p.L;
  const int64_t b = bu, l = tok - bu * (uint32_t)p.L;
  const int i0 = (lane % TPR) * E, hl = lane / TPR;
  const int lo = (int)(task - tok * p.tasks) * p.rpt;
  const int hi = min(lo + p.rpt, p.rq + p.rk);
  F2 cs[P], sn[P];
  bool first = true;
  for (int r0 = lo; r0 < hi; r0 += U) {
    uint4 x1[U], x2[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = r0 + u;
      const bool is_q = r < p.rq;
      const Heads<T>& s = is_q ? p.q : p.k;
      const int h = (is_q ? r : r - p.rq) * RPW + hl;
      x1[u] = x2[u] = make_uint4(0, 0, 0, 0);
      if (r < hi && h < s.H) {
        const T* row = s.x + b * s.xb + (int64_t)h * s.xh + l * s.xs + i0;
        x1[u] = *reinterpret_cast<const uint4*>(row);
        x2[u] = *reinterpret_cast<const uint4*>(row + D / 2);
      }
    }
    if (first) {       // while the first rows are on their way
      float c[E], n[E];
      const int64_t pos = p.pos ? p.pos[b * p.pos_sb + l] : l;
      token_rotation<T, D, E>(pos, p.inv_freq, lane, i0, table[warp], c, n);
#pragma unroll
      for (int v = 0; v < P; ++v) {
        cs[v] = f2(c[2 * v], c[2 * v + 1]);
        sn[v] = f2(n[2 * v], n[2 * v + 1]);
      }
      first = false;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = r0 + u;
      if (r >= hi) break;
      const bool is_q = r < p.rq;
      const Heads<T>& s = is_q ? p.q : p.k;
      const int h = (is_q ? r : r - p.rq) * RPW + hl;
      F2 a1[P], a2[P], ss2 = f2(0.f, 0.f);
      to_pairs<T>(x1[u], a1);
      to_pairs<T>(x2[u], a2);
#pragma unroll
      for (int v = 0; v < P; ++v) ss2 = fma2(a1[v], a1[v], fma2(a2[v], a2[v], ss2));
      float ss, ss_hi;
      split(ss2, ss, ss_hi);
      const float rs = rsqrtf(row_sum<TPR>(ss + ss_hi) * (1.f / D) + p.eps);
      if (h < s.H) {
        const F2 rs2 = f2(rs, rs), minus = f2(-1.f, -1.f);
        F2 w1[P], w2[P], o1[P], o2[P];
        to_pairs<T>(ldg16(s.w + i0), w1);
        to_pairs<T>(ldg16(s.w + D / 2 + i0), w2);
#pragma unroll
        for (int v = 0; v < P; ++v) {
          const F2 n1 = mul2(mul2(a1[v], rs2), w1[v]), n2 = mul2(mul2(a2[v], rs2), w2[v]);
          o1[v] = fma2(n1, cs[v], mul2(mul2(n2, sn[v]), minus));
          o2[v] = fma2(n2, cs[v], mul2(n1, sn[v]));
        }
        T* out = s.o + b * s.ob + (int64_t)h * s.oh + l * s.os + i0;
        stg16(out, from_pairs<T>(o1));
        stg16(out + D / 2, from_pairs<T>(o2));
      }
    }
  }
}

// Forward with few heads: p.nt tokens per warp, a row's heads the query's, then
// the key's.
template <typename T, int TPR>
__global__ void __launch_bounds__(kThreads) fwd_few_kernel(Params<T> p) {
  constexpr int E = Vec<T>::kElems;
  constexpr int P = E / 2;
  constexpr int RPW = 32 / TPR;
  constexpr int D = 2 * E * TPR;
  constexpr int U = kFwdUnroll;
  __shared__ float table[kWarps][kFewRounds * RPW * D];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t task = blockIdx.x * kWarps + warp;
  if ((int64_t)task * p.nt >= p.tokens) return;
  const uint32_t tok0 = task * (uint32_t)p.nt;
  const int nt = min((uint32_t)p.nt, (uint32_t)p.tokens - tok0);
  const int H = p.q.H + p.k.H, rows = nt * H;
  const int i0 = (lane % TPR) * E, hl = lane / TPR;
  fill_rotations<D>(p, tok0, nt, lane, table[warp]);
  for (int r0 = 0; r0 * RPW < rows; r0 += U) {
    uint4 x1[U], x2[U];
    T* out[U];
    const T* w[U];
    const float* rot[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t i = (r0 + u) * RPW + hl;
      x1[u] = x2[u] = make_uint4(0, 0, 0, 0);
      out[u] = nullptr;
      w[u] = nullptr;
      rot[u] = table[warp];
      if (i < (uint32_t)rows) {
        const uint32_t t = i / (uint32_t)H, hh = i - t * H;
        const uint32_t b = (tok0 + t) / (uint32_t)p.L, l = tok0 + t - b * (uint32_t)p.L;
        const bool is_q = hh < (uint32_t)p.q.H;
        const Heads<T>& s = is_q ? p.q : p.k;
        const int64_t h = is_q ? hh : hh - p.q.H;
        const T* row = s.x + (int64_t)b * s.xb + h * s.xh + (int64_t)l * s.xs + i0;
        x1[u] = *reinterpret_cast<const uint4*>(row);
        x2[u] = *reinterpret_cast<const uint4*>(row + D / 2);
        out[u] = s.o + (int64_t)b * s.ob + h * s.oh + (int64_t)l * s.os + i0;
        w[u] = s.w + i0;
        rot[u] = table[warp] + t * D + i0;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      F2 a1[P], a2[P], ss2 = f2(0.f, 0.f);
      to_pairs<T>(x1[u], a1);
      to_pairs<T>(x2[u], a2);
#pragma unroll
      for (int v = 0; v < P; ++v) ss2 = fma2(a1[v], a1[v], fma2(a2[v], a2[v], ss2));
      float ss, ss_hi;
      split(ss2, ss, ss_hi);
      const float rs = rsqrtf(row_sum<TPR>(ss + ss_hi) * (1.f / D) + p.eps);
      if (out[u]) {
        const F2 rs2 = f2(rs, rs), minus = f2(-1.f, -1.f);
        F2 w1[P], w2[P], o1[P], o2[P];
        to_pairs<T>(ldg16(w[u]), w1);
        to_pairs<T>(ldg16(w[u] + D / 2), w2);
#pragma unroll
        for (int v = 0; v < P; ++v) {
          const F2 cs = f2(rot[u][2 * v], rot[u][2 * v + 1]);
          const F2 sn = f2(rot[u][D / 2 + 2 * v], rot[u][D / 2 + 2 * v + 1]);
          const F2 n1 = mul2(mul2(a1[v], rs2), w1[v]), n2 = mul2(mul2(a2[v], rs2), w2[v]);
          o1[v] = fma2(n1, cs, mul2(mul2(n2, sn), minus));
          o2[v] = fma2(n2, cs, mul2(n1, sn));
        }
        stg16(out[u], from_pairs<T>(o1));
        stg16(out[u] + D / 2, from_pairs<T>(o2));
      }
    }
  }
}

// Backward: CTAs [0, q_ctas) stride over the query tasks, the others over the
// key tasks, so a CTA sums one weight gradient; part[cta][D].
template <typename T, int TPR, bool Few>
__device__ __forceinline__ void bwd_side(const Params<T>& p, const Heads<T>& s, bool is_q,
                                         int64_t cta, int64_t ctas, float* table,
                                         F2 (&a1)[2], F2 (&a2)[2]) {
  using V = Quad<T>;
  using Raw = typename V::Raw;
  constexpr int E = 4;
  constexpr int RPW = 32 / TPR;
  constexpr int D = 2 * E * TPR;
  constexpr int U = kBwdUnroll<T>;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int per_tok = is_q ? p.tasks_q : p.tasks_k, rpt = is_q ? p.rpt_q : p.rpt_k;
  const int rounds = is_q ? p.rq : p.rk, few_nt = is_q ? p.nt_q : p.nt_k;
  const int i0 = (lane % TPR) * E, hl = lane / TPR;
  F2 w1[2], w2[2];
  V::to_float(__ldg(reinterpret_cast<const Raw*>(s.w + i0)), w1);
  V::to_float(__ldg(reinterpret_cast<const Raw*>(s.w + D / 2 + i0)), w2);
  const int64_t xstep = RPW * s.xh, dstep = RPW * s.dh, ostep = RPW * s.oh;
  const int64_t tasks = Few ? (p.tokens + few_nt - 1) / few_nt : p.tokens * per_tok;
  const int64_t stride = ctas * kWarps;
  // The next U rounds are loaded while the current ones are worked on, across
  // the border between two tokens too.
  struct Place { int64_t task, pos; int r0, hi; const T* xp; const T* dp; T* op; };
  // Few: a task is U rounds at most; this lane's row of round u is head hs[u] of
  // token ts[u] in every task.
  int ts[U], hs[U];
  if constexpr (Few) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      ts[u] = (u * RPW + hl) / s.H;
      hs[u] = (u * RPW + hl) - ts[u] * s.H;
    }
  }
  struct Token { uint32_t b, l; };
  auto token_of = [&](int64_t task, int t) {
    const uint32_t tok = (uint32_t)task * few_nt + t, b = tok / (uint32_t)p.L;
    return Token{b, tok - b * (uint32_t)p.L};
  };
  auto tokens_of = [&](int64_t task) {
    const int64_t left = p.tokens - task * few_nt;
    return (int)(left < few_nt ? left : few_nt);
  };
  auto enter = [&](Place& at) {          // first rounds of at.task
    if (at.task >= tasks) return;
    if constexpr (Few) {
      at.r0 = 0;
      at.hi = U;
    } else {
      const uint32_t task = (uint32_t)at.task;
      const uint32_t tok = task / (uint32_t)per_tok, bu = tok / (uint32_t)p.L;
      const int64_t b = bu, l = tok - bu * (uint32_t)p.L;
      at.r0 = (int)(task - tok * per_tok) * rpt;
      at.hi = min(at.r0 + rpt, rounds);
      const int64_t h0 = (int64_t)at.r0 * RPW + hl;
      at.xp = s.x + b * s.xb + h0 * s.xh + l * s.xs + i0;
      at.dp = s.d + b * s.db + h0 * s.dh + l * s.ds + i0;
      at.op = s.o + b * s.ob + h0 * s.oh + l * s.os + i0;
      at.pos = p.pos ? p.pos[b * p.pos_sb + l] : l;
    }
  };
  auto load = [&](Place& at, Raw (&x1)[U], Raw (&x2)[U], Raw (&d1)[U], Raw (&d2)[U]) {
    const int nt = Few && at.task < tasks ? tokens_of(at.task) : 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      x1[u] = x2[u] = d1[u] = d2[u] = V::zero();
      bool in;
      if constexpr (Few) {
        in = ts[u] < nt;
        if (in) {
          const Token k = token_of(at.task, ts[u]);
          at.xp = s.x + (int64_t)k.b * s.xb + (int64_t)hs[u] * s.xh + (int64_t)k.l * s.xs + i0;
          at.dp = s.d + (int64_t)k.b * s.db + (int64_t)hs[u] * s.dh + (int64_t)k.l * s.ds + i0;
        }
      } else {
        in = at.task < tasks && at.r0 + u < at.hi && (at.r0 + u) * RPW + hl < s.H;
      }
      if (in) {
        x1[u] = *reinterpret_cast<const Raw*>(at.xp);
        x2[u] = *reinterpret_cast<const Raw*>(at.xp + D / 2);
        d1[u] = *reinterpret_cast<const Raw*>(at.dp);
        d2[u] = *reinterpret_cast<const Raw*>(at.dp + D / 2);
      }
      if constexpr (!Few) {
        at.xp += xstep;
        at.dp += dstep;
      }
    }
  };
  Place next{};
  next.task = cta * kWarps + warp;
  Raw nx1[U], nx2[U], nd1[U], nd2[U];
  enter(next);
  load(next, nx1, nx2, nd1, nd2);
  F2 cs[2], sn[2], ns[2];
  auto set_rotation = [&](const float (&c)[E], const float (&n)[E]) {
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      cs[v] = f2(c[2 * v], c[2 * v + 1]);
      sn[v] = f2(n[2 * v], n[2 * v + 1]);
      ns[v] = f2(-n[2 * v], -n[2 * v + 1]);
    }
  };
  int64_t done = -1;                     // the task whose angles are held
  while (next.task < tasks) {
    Raw x1[U], x2[U], d1[U], d2[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      x1[u] = nx1[u]; x2[u] = nx2[u]; d1[u] = nd1[u]; d2[u] = nd2[u];
    }
    const int r0 = next.r0, hi = next.hi;
    const int64_t task = next.task, pos = next.pos;
    T* op = next.op;
    next.r0 += U;
    next.op += U * ostep;
    if (next.r0 >= hi) {
      next.task += stride;
      enter(next);
    }
    load(next, nx1, nx2, nd1, nd2);
    const int nt = Few ? tokens_of(task) : 0;
    if (task != done) {
      if constexpr (Few) {
        fill_rotations<D>(p, (uint32_t)task * few_nt, nt, lane, table);
      } else {
        float c[E], n[E];
        token_rotation<T, D, E>(pos, p.inv_freq, lane, i0, table, c, n);
        set_rotation(c, n);
      }
      done = task;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (r0 + u >= hi) break;
      bool in;
      if constexpr (Few) {
        if (u * RPW >= nt * s.H) break;
        in = ts[u] < nt;
        if (in) {
          const Token k = token_of(task, ts[u]);
          op = s.o + (int64_t)k.b * s.ob + (int64_t)hs[u] * s.oh + (int64_t)k.l * s.os + i0;
          const float* rot = table + ts[u] * D + i0;
          float c[E], n[E];
#pragma unroll
          for (int e = 0; e < E; ++e) {
            c[e] = rot[e];
            n[e] = rot[D / 2 + e];
          }
          set_rotation(c, n);
        } else {
          const float z[E] = {};
          set_rotation(z, z);
        }
      } else {
        in = (r0 + u) * RPW + hl < s.H;
      }
      F2 xv1[2], xv2[2], y1[2], y2[2], g1[2], g2[2], gw1[2], gw2[2];
      F2 ss2 = f2(0.f, 0.f), dot2 = f2(0.f, 0.f);
      V::to_float(x1[u], xv1);
      V::to_float(x2[u], xv2);
      V::to_float(d1[u], y1);
      V::to_float(d2[u], y2);
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        g1[v] = fma2(y1[v], cs[v], mul2(y2[v], sn[v]));
        g2[v] = fma2(y2[v], cs[v], mul2(y1[v], ns[v]));
        gw1[v] = mul2(g1[v], w1[v]);
        gw2[v] = mul2(g2[v], w2[v]);
        ss2 = fma2(xv1[v], xv1[v], fma2(xv2[v], xv2[v], ss2));
        dot2 = fma2(gw1[v], xv1[v], fma2(gw2[v], xv2[v], dot2));
      }
      float ss, dot, hi_ss, hi_dot;
      split(ss2, ss, hi_ss);
      split(dot2, dot, hi_dot);
      ss += hi_ss;
      dot += hi_dot;
      row_sum2<TPR>(ss, dot);
      // dx = rstd w g - x rstd^3 mean(x w g)
      const float rs = rsqrtf(ss * (1.f / D) + p.eps);
      const float c = -(dot * rs * (1.f / D)) * rs * rs;
      const F2 rs2 = f2(rs, rs), c2 = f2(c, c);
      if (in) {
        F2 o1[2], o2[2];
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          a1[v] = fma2(g1[v], mul2(xv1[v], rs2), a1[v]);
          a2[v] = fma2(g2[v], mul2(xv2[v], rs2), a2[v]);
          o1[v] = fma2(xv1[v], c2, mul2(gw1[v], rs2));
          o2[v] = fma2(xv2[v], c2, mul2(gw2[v], rs2));
        }
        *reinterpret_cast<Raw*>(op) = V::from_float(o1);
        *reinterpret_cast<Raw*>(op + D / 2) = V::from_float(o2);
      }
      if constexpr (!Few) op += ostep;
    }
  }
}

template <typename T, int TPR>
__global__ void __launch_bounds__(kThreads, kBwdCtasPerSm)
bwd_kernel(Params<T> p, int q_ctas, float* part) {
  constexpr int E = 4;
  constexpr int RPW = 32 / TPR;
  constexpr int D = 2 * E * TPR;
  // angles of the warps' tokens (at most U * RPW of them), then sums
  __shared__ float red[kWarps][kBwdUnroll<T> * RPW * D];
  cudaTriggerProgrammaticLaunchCompletion();  // the sum's CTAs may take free SMs
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool is_q = (int)blockIdx.x < q_ctas;
  const Heads<T>& s = is_q ? p.q : p.k;
  const int64_t cta = is_q ? blockIdx.x : blockIdx.x - q_ctas;
  const int64_t ctas = is_q ? q_ctas : gridDim.x - q_ctas;
  const int i0 = (lane % TPR) * E;
  F2 a1[2], a2[2];
#pragma unroll
  for (int v = 0; v < 2; ++v) a1[v] = a2[v] = f2(0.f, 0.f);
  if ((is_q ? p.nt_q : p.nt_k) > 1)
    bwd_side<T, TPR, true>(p, s, is_q, cta, ctas, red[warp], a1, a2);
  else
    bwd_side<T, TPR, false>(p, s, is_q, cta, ctas, red[warp], a1, a2);
  __syncwarp();
  float s1[E], s2[E];
#pragma unroll
  for (int v = 0; v < 2; ++v) {
    split(a1[v], s1[2 * v], s1[2 * v + 1]);
    split(a2[v], s2[2 * v], s2[2 * v + 1]);
  }
  // rows of the warp, then warps
#pragma unroll
  for (int o = TPR; o < 32; o <<= 1) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      s1[e] += __shfl_xor_sync(0xffffffffu, s1[e], o);
      s2[e] += __shfl_xor_sync(0xffffffffu, s2[e], o);
    }
  }
  if (lane < TPR) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      red[warp][i0 + e] = s1[e];
      red[warp][D / 2 + i0 + e] = s2[e];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < D; i += kThreads) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) v += red[w][i];
    part[(int64_t)blockIdx.x * D + i] = v;
  }
}

// dw of the query side (y = 0) and the key side (y = 1; y = 0 when there are
// keys only: first = 1) from the CTAs' partials, in a fixed order.  The partials
// may still be written when this kernel starts: no __restrict__ on them, so that
// they are not read through the read-only path.
constexpr int kSumWarps = 32;

template <typename T>
__global__ void __launch_bounds__(kSumWarps * 32)
sum_kernel(int D, int q_ctas, int ctas, int first, const float* part, T* dwq, T* dwk) {
  __shared__ float red[kSumWarps][33];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  cudaGridDependencySynchronize();
  const bool keys = blockIdx.y + first > 0;
  const int lo = keys ? q_ctas : 0, hi = keys ? ctas : q_ctas;
  const int col = blockIdx.x * 32 + lane;
  float v = 0.f;
  if (col < D)
    for (int c = lo + warp; c < hi; c += kSumWarps) v += part[(int64_t)c * D + col];
  red[warp][lane] = v;
  __syncthreads();
  if (warp == 0 && col < D) {
    for (int w = 1; w < kSumWarps; ++w) v += red[w][lane];
    (keys ? dwk : dwq)[col] = from_f32<T>(v);
  }
}

}  // namespace qknorm
}  // namespace esa
