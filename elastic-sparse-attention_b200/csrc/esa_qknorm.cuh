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
// A row is held by D / (2 E) threads (E elements per 16-byte vector): thread t
// owns elements [tE, tE + E) and the same of the second half, so the rotation
// needs no exchange.  A warp takes several heads of one token, so the angles
// are formed once per token and thread.  HBM-bound: every element is read and
// written once; rstd is formed again in the backward instead of being kept.
#pragma once
#include "esa_common.cuh"

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
  int hpt;                            // heads per warp task
  int cq, ck;                         // tasks per token of the query / key heads
};

// cos and sin of p * f: the product in float64 (p and f are exact there), in
// turns, so that far positions lose nothing to the reduction.
__device__ __forceinline__ void rotation(int64_t p, float f, float& c, float& s) {
  double t = (double)p * (double)f * 0.15915494309189533577;   // 1 / (2 pi)
  t -= rint(t);
  sincospif((float)(2.0 * t), &s, &c);
}

template <int TPR>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = TPR / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;

template <typename T, int TPR>
__global__ void __launch_bounds__(kThreads) fwd_kernel(Params<T> p) {
  using V = Vec<T>;
  constexpr int E = V::kElems;
  constexpr int RPW = 32 / TPR;               // rows a warp holds at once
  constexpr int D = 2 * E * TPR;
  const int lane = threadIdx.x & 31;
  const int64_t task = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  const int64_t tok = task / (p.cq + p.ck);
  if (tok >= p.tokens) return;
  int c = (int)(task - tok * (p.cq + p.ck));
  const bool is_q = c < p.cq;
  const Heads<T>& s = is_q ? p.q : p.k;
  if (!is_q) c -= p.cq;
  const int64_t b = tok / p.L, l = tok - b * p.L;
  const int i0 = (lane % TPR) * E;
  const int64_t pos = p.pos ? p.pos[b * p.pos_sb + l] : l;
  float cs[E], sn[E], w1[E], w2[E];
#pragma unroll
  for (int e = 0; e < E; ++e) rotation(pos, p.inv_freq[i0 + e], cs[e], sn[e]);
  V::to_float(ldg16(s.w + i0), w1);
  V::to_float(ldg16(s.w + D / 2 + i0), w2);
  const int h1 = min((c + 1) * p.hpt, s.H);
  for (int h0 = c * p.hpt; h0 < h1; h0 += RPW) {
    const int h = h0 + lane / TPR;
    const bool in = h < h1;
    float x1[E], x2[E], ss = 0.f;
    const T* row = s.x + b * s.xb + (int64_t)h * s.xh + l * s.xs;
    if (in) {
      V::to_float(*reinterpret_cast<const uint4*>(row + i0), x1);
      V::to_float(*reinterpret_cast<const uint4*>(row + D / 2 + i0), x2);
#pragma unroll
      for (int e = 0; e < E; ++e) ss = fmaf(x1[e], x1[e], fmaf(x2[e], x2[e], ss));
    }
    const float rs = rsqrtf(row_sum<TPR>(ss) * (1.f / D) + p.eps);
    if (in) {
      float o1[E], o2[E];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float n1 = x1[e] * rs * w1[e], n2 = x2[e] * rs * w2[e];
        o1[e] = n1 * cs[e] - n2 * sn[e];
        o2[e] = n2 * cs[e] + n1 * sn[e];
      }
      T* out = s.o + b * s.ob + (int64_t)h * s.oh + l * s.os;
      stg16(out + i0, V::from_float(o1));
      stg16(out + D / 2 + i0, V::from_float(o2));
    }
  }
}

// Backward: CTAs [0, q_ctas) stride over the query tasks, the others over the
// key tasks, so a CTA sums one weight gradient; part[cta][D].
template <typename T, int TPR>
__global__ void __launch_bounds__(kThreads) bwd_kernel(Params<T> p, int q_ctas, float* part) {
  using V = Vec<T>;
  constexpr int E = V::kElems;
  constexpr int RPW = 32 / TPR;
  constexpr int D = 2 * E * TPR;
  __shared__ float red[kWarps][D];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool is_q = (int)blockIdx.x < q_ctas;
  const Heads<T>& s = is_q ? p.q : p.k;
  const int chunks = is_q ? p.cq : p.ck;
  const int64_t cta = is_q ? blockIdx.x : blockIdx.x - q_ctas;
  const int64_t ctas = is_q ? q_ctas : gridDim.x - q_ctas;
  const int i0 = (lane % TPR) * E;
  float w1[E], w2[E], a1[E], a2[E];
  V::to_float(ldg16(s.w + i0), w1);
  V::to_float(ldg16(s.w + D / 2 + i0), w2);
#pragma unroll
  for (int e = 0; e < E; ++e) a1[e] = a2[e] = 0.f;
  const int64_t tasks = p.tokens * chunks;
  for (int64_t task = cta * kWarps + warp; task < tasks; task += ctas * kWarps) {
    const int64_t tok = task / chunks;
    const int c = (int)(task - tok * chunks);
    const int64_t b = tok / p.L, l = tok - b * p.L;
    const int64_t pos = p.pos ? p.pos[b * p.pos_sb + l] : l;
    float cs[E], sn[E];
#pragma unroll
    for (int e = 0; e < E; ++e) rotation(pos, p.inv_freq[i0 + e], cs[e], sn[e]);
    const int h1 = min((c + 1) * p.hpt, s.H);
    for (int h0 = c * p.hpt; h0 < h1; h0 += RPW) {
      const int h = h0 + lane / TPR;
      const bool in = h < h1;
      float x1[E], x2[E], g1[E], g2[E], ss = 0.f, dot = 0.f;
      if (in) {
        const T* row = s.x + b * s.xb + (int64_t)h * s.xh + l * s.xs;
        const T* drow = s.d + b * s.db + (int64_t)h * s.dh + l * s.ds;
        float d1[E], d2[E];
        V::to_float(*reinterpret_cast<const uint4*>(row + i0), x1);
        V::to_float(*reinterpret_cast<const uint4*>(row + D / 2 + i0), x2);
        V::to_float(*reinterpret_cast<const uint4*>(drow + i0), d1);
        V::to_float(*reinterpret_cast<const uint4*>(drow + D / 2 + i0), d2);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          g1[e] = d1[e] * cs[e] + d2[e] * sn[e];
          g2[e] = d2[e] * cs[e] - d1[e] * sn[e];
          ss = fmaf(x1[e], x1[e], fmaf(x2[e], x2[e], ss));
          dot = fmaf(g1[e] * w1[e], x1[e], fmaf(g2[e] * w2[e], x2[e], dot));
        }
      }
      ss = row_sum<TPR>(ss);
      dot = row_sum<TPR>(dot);
      const float rs = rsqrtf(ss * (1.f / D) + p.eps);
      if (in) {
        const float m = dot * rs * (1.f / D);
        float o1[E], o2[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float h1v = x1[e] * rs, h2v = x2[e] * rs;
          a1[e] = fmaf(g1[e], h1v, a1[e]);
          a2[e] = fmaf(g2[e], h2v, a2[e]);
          o1[e] = rs * (w1[e] * g1[e] - h1v * m);
          o2[e] = rs * (w2[e] * g2[e] - h2v * m);
        }
        T* out = s.o + b * s.ob + (int64_t)h * s.oh + l * s.os;
        stg16(out + i0, V::from_float(o1));
        stg16(out + D / 2 + i0, V::from_float(o2));
      }
    }
  }
  // rows of the warp, then warps
#pragma unroll
  for (int o = TPR; o < 32; o <<= 1) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      a1[e] += __shfl_xor_sync(0xffffffffu, a1[e], o);
      a2[e] += __shfl_xor_sync(0xffffffffu, a2[e], o);
    }
  }
  if (lane < TPR) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      red[warp][i0 + e] = a1[e];
      red[warp][D / 2 + i0 + e] = a2[e];
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
// keys only: first = 1) from the CTAs' partials, in a fixed order.
constexpr int kSumWarps = 32;

template <typename T>
__global__ void __launch_bounds__(kSumWarps * 32)
sum_kernel(int D, int q_ctas, int ctas, int first, const float* __restrict__ part, T* dwq,
           T* dwk) {
  __shared__ float red[kSumWarps][33];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
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
