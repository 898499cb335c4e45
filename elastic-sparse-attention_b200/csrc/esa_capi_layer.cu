// extern "C" entry points of include/esa_layer.h: token embedding and its
// gradient, per-head query / key norm with the rotary embedding, activations
// kept in 8 bits.  (RMSNorm, rotary embedding and SwiGLU are in esa_capi.cu.)
#include <algorithm>
#include <cmath>

#include "esa_layer.h"
#include "esa_embed.cuh"
#include "esa_host.h"
#include "esa_pack8.cuh"
#include "esa_qknorm.cuh"

namespace {

using namespace esa::host;

size_t align256(size_t x) { return (x + 255) / 256 * 256; }

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// ---------------------------------------------------------------------------
// Token embedding.
// ---------------------------------------------------------------------------
namespace em = esa::embed;

constexpr int64_t kMaxTokens = int64_t(1) << 30;
constexpr int64_t kMaxVocab = (int64_t(1) << 27) - 1;   // three digits of 9 bits, one key spare

int check_embedding(const char* what, int32_t dtype, int32_t id_bytes, int64_t n, int64_t vocab,
                    int32_t dim, const void* ids, float scale) {
  if (int rc = check_rows_op(what, dtype, n, dim)) return rc;
  if (id_bytes != 4 && id_bytes != 8)
    return fail(ESA_ERR_INVALID, "%s: id_bytes %d (4 or 8)", what, id_bytes);
  if (vocab < 1) return fail(ESA_ERR_INVALID, "%s: vocab must be >= 1", what);
  if (vocab > kMaxVocab || n > kMaxTokens)
    return fail(ESA_ERR_UNSUPPORTED, "%s: more than 2^27 - 1 rows or 2^30 tokens", what);
  if (!std::isfinite(scale)) return fail(ESA_ERR_INVALID, "%s: scale must be finite", what);
  if (n > 0 && (!ids || reinterpret_cast<uintptr_t>(ids) % id_bytes))
    return fail(ESA_ERR_INVALID, "%s: null or misaligned ids", what);
  return ESA_OK;
}

// Geometry and workspace of the sorted gradient.
struct GradPlan {
  int key_bits;              // keys are 0 .. vocab
  int passes, bits;          // digits of the key, bits per digit
  int tile;                  // keys per sorting CTA
  int64_t tiles, pieces;
  size_t keys[2], rows[2], hist, part, owners, counter, bytes;   // offsets
};

GradPlan grad_plan(int64_t n, int64_t vocab, int32_t dim) {
  GradPlan g;
  g.key_bits = 1;
  while ((vocab >> g.key_bits) != 0) ++g.key_bits;
  g.passes = (int)ceil_div(g.key_bits, em::kRadixBits);
  g.bits = (int)ceil_div(g.key_bits, g.passes);
  g.tile = em::kSortTile;
  while (ceil_div(n, g.tile) > em::kSortTiles &&
         (g.tile < 2 * em::kSortTile || ceil_div(n, g.tile) > em::kSortMaxTiles))
    g.tile += em::kSortTile;
  g.tiles = ceil_div(n, g.tile);
  g.pieces = ceil_div(n, em::piece_len(n, dim));
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at += align256(bytes);
    return o;
  };
  for (int i = 0; i < 2; ++i) {
    g.keys[i] = take(n * 4);
    g.rows[i] = take(n * 4);
  }
  g.hist = take(g.tiles * em::kRadix * 4);
  g.owners = take(g.pieces * sizeof(uint2));
  g.counter = take(4);
  g.part = take((size_t)g.pieces * 2 * dim * sizeof(float));
  g.bytes = at;
  return g;
}

template <typename T>
int embedding_grad(int64_t n, int64_t vocab, int32_t dim, const em::Ids& ids, const void* dy,
                   float scale, int64_t pad, void* dweight, char* ws, int* err, cudaStream_t s) {
  const uint32_t vpr = dim / esa::Vec<T>::kElems;
  if (vpr > 32 * 65535) return fail(ESA_ERR_UNSUPPORTED, "esa_embedding_backward: dim %d too large", dim);
  if (n <= em::direct_max(dim)) {
    auto direct = [&](auto nv) {
      constexpr int NV = decltype(nv)::value;
      // about eight CTAs per SM over the vocabulary, 32 rows of it at most
      const unsigned chunks = (unsigned)ceil_div(vpr, 32 * NV);
      const int R = (int)std::min<int64_t>(32, ceil_div(vocab * chunks, 148 * 8));
      em::grad_direct_kernel<T, NV>
          <<<dim3((unsigned)ceil_div(vocab, R), chunks), em::kDirectThreads, 0, s>>>(
              (int)n, vocab, R, vpr, ids, static_cast<const T*>(dy), scale, pad,
              static_cast<T*>(dweight), err);
      return check_launch("esa_embedding_backward");
    };
    if (vpr > 64) return direct(std::integral_constant<int, 4>{});
    return direct(std::integral_constant<int, 1>{});
  }
  const GradPlan g = grad_plan(n, vocab, dim);
  uint32_t* keys[2];
  uint32_t* rows[2];
  for (int i = 0; i < 2; ++i) {
    keys[i] = reinterpret_cast<uint32_t*>(ws + g.keys[i]);
    rows[i] = reinterpret_cast<uint32_t*>(ws + g.rows[i]);
  }
  int* counter = reinterpret_cast<int*>(ws + g.counter);
  int last = 0;                          // which buffer holds the sorted pairs
  if (n <= em::kSmallMax) {
    em::SmallSort p;
    p.vocab = vocab;
    p.pad = pad;
    p.ids = ids;
    p.n = (int)n;
    p.passes = (int)ceil_div(g.key_bits, em::kSmallBits);
    p.bits = (int)ceil_div(g.key_bits, p.passes);
    p.out_keys = keys[0];
    p.out_rows = rows[0];
    p.counter = counter;
    p.err = err;
    em::sort_small_kernel<<<1, em::kSmallThreads, 0, s>>>(p);
    if (int rc = check_launch("esa_embedding_backward (sort)")) return rc;
  } else {
    em::SortPass p;
    p.n = n;
    p.vocab = vocab;
    p.pad = pad;
    p.ids = ids;
    p.keys = p.rows = nullptr;
    p.bits = g.bits;
    p.tile = g.tile;
    p.hist = reinterpret_cast<uint32_t*>(ws + g.hist);
    p.counter = counter;
    p.err = err;
    for (int i = 0; i < g.passes; ++i) {
      p.shift = i * g.bits;
      p.out_keys = keys[i & 1];
      p.out_rows = rows[i & 1];
      const dim3 grid((unsigned)g.tiles), block(em::kSortThreads);
      if (i == 0) {
        em::sort_hist_kernel<<<grid, block, 0, s>>>(p);
        if (int rc = check_launch("esa_embedding_backward (histogram)")) return rc;
      } else if (int rc = launch_after("esa_embedding_backward (histogram)", em::sort_hist_kernel,
                                       grid, block, s, p)) {
        return rc;
      }
      if (int rc = launch_after("esa_embedding_backward (sort)", em::sort_scatter_kernel, grid,
                                block, s, p))
        return rc;
      p.keys = p.out_keys;
      p.rows = p.out_rows;
      last = i & 1;
    }
  }
  em::GradParams q;
  q.n = n;
  q.vocab = vocab;
  q.vpr = vpr;
  q.keys = keys[last];
  q.rows = rows[last];
  q.scale = scale;
  q.part = reinterpret_cast<float*>(ws + g.part);
  q.counter = counter;
  q.owners = reinterpret_cast<uint2*>(ws + g.owners);
  q.pieces = g.pieces;
  q.zero_blocks = (int)ceil_div(vocab, em::kZeroRows);
  q.piece = em::piece_len(n, dim);
  auto pieces = [&](auto piece, auto threads) {
    constexpr int P = decltype(piece)::value, TH = decltype(threads)::value;
    q.ychunks = (int)ceil_div(vpr, TH);
    const int64_t ctas = (q.zero_blocks + g.pieces) * q.ychunks;
    if (ctas > INT32_MAX)
      return fail(ESA_ERR_UNSUPPORTED, "esa_embedding_backward: too many tokens");
    return launch_after("esa_embedding_backward (sums)", em::grad_pieces_kernel<T, P, TH>,
                        dim3((unsigned)ctas), dim3(TH), s, q, static_cast<const T*>(dy),
                        static_cast<T*>(dweight));
  };
  using std::integral_constant;
  int rc;
  if (em::narrow_rows(dim))
    rc = pieces(integral_constant<int, 16>{}, integral_constant<int, 32>{});
  else if (q.piece == 16)
    rc = pieces(integral_constant<int, 16>{}, integral_constant<int, 128>{});
  else if (q.piece == 32)
    rc = pieces(integral_constant<int, 32>{}, integral_constant<int, 128>{});
  else
    rc = pieces(integral_constant<int, 64>{}, integral_constant<int, 128>{});
  if (rc) return rc;
  return launch_after("esa_embedding_backward (join)", em::grad_join_kernel<T>, dim3(148 * 8),
                      dim3(em::kJoinWarps * 32), s, q, static_cast<T*>(dweight));
}

// ---------------------------------------------------------------------------
// Query / key norm with the rotary embedding.
// ---------------------------------------------------------------------------
namespace qk = esa::qknorm;

constexpr int kQkBwdCtas = 148 * qk::kBwdCtasPerSm;   // fixed, so the weight gradients' sums do not depend on the GPU

int check_qk(const char* what, int32_t dtype, int32_t batch, int64_t seq_len, int32_t head_dim,
             int32_t num_q_heads, int32_t num_k_heads, int64_t pos_stride, float eps) {
  if (dtype != ESA_DTYPE_F32 && dtype != ESA_DTYPE_BF16 && dtype != ESA_DTYPE_F16)
    return fail(ESA_ERR_INVALID, "%s: unknown dtype %d", what, dtype);
  if (batch < 0 || seq_len < 0 || num_q_heads < 0 || num_k_heads < 0 || pos_stride < 0)
    return fail(ESA_ERR_INVALID, "%s: negative size", what);
  const int per = 2 * (16 / elem_size(dtype));     // elements a thread owns
  if (head_dim < per || head_dim > 16 * per || (head_dim & (head_dim - 1)))
    return fail(ESA_ERR_UNSUPPORTED, "%s: head_dim %d (a power of two in [%d, %d])", what, head_dim,
                per, 16 * per);
  if ((int64_t)batch * seq_len > INT32_MAX || num_q_heads > 65535 || num_k_heads > 65535)
    return fail(ESA_ERR_UNSUPPORTED, "%s: too many positions or heads", what);
  if (!(eps >= 0.f) || !std::isfinite(eps))
    return fail(ESA_ERR_INVALID, "%s: eps must be finite and not negative", what);
  return ESA_OK;
}

template <typename T>
int set_heads(qk::Heads<T>& s, const char* name, const esa_tensor_t& x, const esa_tensor_t* d,
              const esa_tensor_t& o, const void* w, int H) {
  s = qk::Heads<T>{};
  s.H = H;
  if (H == 0) return ESA_OK;
  const int es = sizeof(T);
  if (int rc = check_tensor(name, x, es)) return rc;
  if (d)
    if (int rc = check_tensor(name, *d, es)) return rc;
  if (int rc = check_tensor(name, o, es)) return rc;
  if (!w || !aligned16(w)) return fail(ESA_ERR_INVALID, "%s weight: null or misaligned pointer", name);
  s.x = static_cast<const T*>(x.data);
  s.xb = x.stride_b; s.xh = x.stride_h; s.xs = x.stride_s;
  if (d) {
    s.d = static_cast<const T*>(d->data);
    s.db = d->stride_b; s.dh = d->stride_h; s.ds = d->stride_s;
  }
  s.o = static_cast<T*>(o.data);
  s.ob = o.stride_b; s.oh = o.stride_h; s.os = o.stride_s;
  s.w = static_cast<const T*>(w);
  return ESA_OK;
}

// f(std::integral_constant<int, threads per row>) for a power of two in [Least, 16 * Least]
template <int Least, typename F>
int by_threads_per_row(int tpr, F&& f) {
  if (tpr == Least) return f(std::integral_constant<int, Least>{});
  if (tpr == 2 * Least) return f(std::integral_constant<int, 2 * Least>{});
  if (tpr == 4 * Least) return f(std::integral_constant<int, 4 * Least>{});
  if (tpr == 8 * Least) return f(std::integral_constant<int, 8 * Least>{});
  return f(std::integral_constant<int, 16 * Least>{});
}

// Rounds per warp task: all of a token's once there are tokens enough for 16
// warps per SM, fewer (down to one) for few tokens.
int rounds_per_task(int rounds, int64_t tokens) {
  if (rounds == 0) return 1;
  const int64_t tasks = std::max<int64_t>(1, std::min<int64_t>(rounds, ceil_div(148 * 16, tokens)));
  return (int)ceil_div(rounds, tasks);
}

// Tokens of a task that takes several because a token's heads fill less than
// one of its rounds, or a quarter of them (1: they fill more).  With half of
// them filled a task of one token is faster (16 / 4 heads of 128, bf16
// backward, 9910 tokens: 43 against 54 us).  No more than leaves 16 warps per
// SM a task.
int tokens_per_task(int heads, int rows_per_warp, int rounds, int64_t tokens) {
  if (heads == 0 || (heads >= rows_per_warp && rounds < 4 * ceil_div(heads, rows_per_warp))) return 1;
  return (int)std::max<int64_t>(1, std::min<int64_t>(rounds * rows_per_warp / heads,
                                                     tokens / (148 * 16)));
}

template <typename T>
void set_tasks(qk::Params<T>& p, int rows_per_warp) {
  p.nt = tokens_per_task(p.q.H + p.k.H, rows_per_warp, qk::kFewRounds, p.tokens);
  p.nt_q = tokens_per_task(p.q.H, rows_per_warp, qk::kBwdUnroll<T>, p.tokens);
  p.nt_k = tokens_per_task(p.k.H, rows_per_warp, qk::kBwdUnroll<T>, p.tokens);
  p.rq = (int)ceil_div(p.q.H, rows_per_warp);
  p.rk = (int)ceil_div(p.k.H, rows_per_warp);
  p.rpt = rounds_per_task(p.rq + p.rk, p.tokens);
  p.tasks = (int)ceil_div(p.rq + p.rk, p.rpt);
  p.rpt_q = rounds_per_task(p.rq, p.tokens);
  p.rpt_k = rounds_per_task(p.rk, p.tokens);
  p.tasks_q = (int)ceil_div(p.rq, p.rpt_q);
  p.tasks_k = (int)ceil_div(p.rk, p.rpt_k);
}

int qk_bwd_ctas(int64_t tokens, int32_t hq, int32_t hk) {
  return (int)std::max<int64_t>(2, std::min<int64_t>(kQkBwdCtas, ceil_div(tokens * (hq + hk), qk::kWarps)));
}

// Share of the CTAs that the query heads get (at least one for each side
// present): by the loop steps of the two sides, which take about as long
// whether their U rounds are full or not.
template <typename T>
int qk_q_ctas(const qk::Params<T>& p, int ctas) {
  if (p.k.H == 0) return ctas;
  if (p.q.H == 0) return 0;
  auto steps = [&](int nt, int tasks, int rpt) {
    return nt > 1 ? ceil_div(p.tokens, nt) : p.tokens * tasks * ceil_div(rpt, qk::kBwdUnroll<T>);
  };
  const int64_t q = steps(p.nt_q, p.tasks_q, p.rpt_q), k = steps(p.nt_k, p.tasks_k, p.rpt_k);
  return (int)std::max<int64_t>(1, std::min<int64_t>(ctas - 1, ctas * q / (q + k)));
}

// ---------------------------------------------------------------------------
// 8-bit rows.
// ---------------------------------------------------------------------------
namespace p8 = esa::pack8;

int check_pack(const char* what, int32_t dtype, int32_t format, int64_t n_rows, int32_t dim) {
  if (int rc = check_rows_op(what, dtype, n_rows, dim)) return rc;
  if (format != ESA_PACK_INT8 && format != ESA_PACK_E4M3)
    return fail(ESA_ERR_INVALID, "%s: unknown 8-bit format %d", what, format);
  if (dim > (1 << 28)) return fail(ESA_ERR_UNSUPPORTED, "%s: dim %d too large", what, dim);
  const int64_t units = ceil_div(dim / (16 / elem_size(dtype)), 32);   // of 32 vectors, per row
  if (n_rows > (int64_t(1) << 31) / units)
    return fail(ESA_ERR_UNSUPPORTED, "%s: too many rows", what);
  return ESA_OK;
}

template <typename F>
int by_format(int32_t format, F&& f) {
  if (format == ESA_PACK_INT8) return f(std::integral_constant<int, p8::kInt8>{});
  return f(std::integral_constant<int, p8::kE4m3>{});
}

// Grid of the kernels whose warps take K * 32 vectors of a row.
unsigned part_grid(int64_t rows, int32_t dim, int elems, int K) {
  return (unsigned)ceil_div(rows * ceil_div(dim / elems, 32 * K), p8::kWarps);
}

// f(vectors per lane, warps per row) for a row of `vecs` 16-byte vectors: at
// most four per lane, as few warps as hold the row.
template <typename F>
int by_row_shape(int vecs, F&& f) {
  using std::integral_constant;
  if (vecs <= 32) return f(integral_constant<int, 1>{}, integral_constant<int, 1>{});
  if (vecs <= 64) return f(integral_constant<int, 2>{}, integral_constant<int, 1>{});
  if (vecs <= 128) return f(integral_constant<int, 4>{}, integral_constant<int, 1>{});
  if (vecs <= 256) return f(integral_constant<int, 4>{}, integral_constant<int, 2>{});
  if (vecs <= 512) return f(integral_constant<int, 4>{}, integral_constant<int, 4>{});
  return f(integral_constant<int, 4>{}, integral_constant<int, 8>{});
}

int check_norm_rows(const char* what, int32_t dtype, int64_t n_rows, int32_t dim, float eps) {
  if (dim > 1024 * (16 / elem_size(dtype)))
    return fail(ESA_ERR_UNSUPPORTED, "%s: dim %d too large", what, dim);
  if (n_rows > INT32_MAX)
    return fail(ESA_ERR_UNSUPPORTED, "%s: too many rows", what);
  if (!(eps >= 0.f) || !std::isfinite(eps))
    return fail(ESA_ERR_INVALID, "%s: eps must be finite and not negative", what);
  return ESA_OK;
}

}  // namespace

extern "C" {

int esa_embedding_forward(int32_t dtype, int32_t id_bytes, int64_t n_tokens, int64_t vocab,
                          int32_t dim, const void* ids, const void* weight, float scale, void* out,
                          void* stream) {
  if (int rc = check_embedding("esa_embedding_forward", dtype, id_bytes, n_tokens, vocab, dim, ids,
                               scale))
    return rc;
  if (n_tokens == 0) return ESA_OK;
  if (!weight || !out || !aligned16(weight) || !aligned16(out))
    return fail(ESA_ERR_INVALID, "esa_embedding_forward: null or misaligned pointer");
  const int64_t vpr = dim / (16 / elem_size(dtype));
  const int64_t ctas = ceil_div(n_tokens * vpr, em::kLookupThreads * em::kLookupUnroll);
  if (ctas > INT32_MAX)
    return fail(ESA_ERR_UNSUPPORTED, "esa_embedding_forward: output too large");
  int* err = nullptr;
  if (int rc = device_error_word(&err)) return rc;
  const em::Ids src{ids, id_bytes == 8};
  return by_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    em::lookup_kernel<T><<<(unsigned)ctas, em::kLookupThreads, 0, (cudaStream_t)stream>>>(
        n_tokens, vocab, (uint32_t)vpr, src, static_cast<const T*>(weight), scale,
        static_cast<T*>(out), err);
    return check_launch("esa_embedding_forward");
  });
}

size_t esa_embedding_backward_workspace_size(int64_t n_tokens, int64_t vocab, int32_t dim) {
  if (n_tokens <= em::direct_max(dim) || n_tokens > kMaxTokens || vocab < 1 || vocab > kMaxVocab ||
      dim < 1)
    return 0;
  return grad_plan(n_tokens, vocab, dim).bytes;
}

int esa_embedding_backward(int32_t dtype, int32_t id_bytes, int64_t n_tokens, int64_t vocab,
                           int32_t dim, const void* ids, const void* dy, float scale,
                           int64_t padding_idx, void* dweight, void* workspace,
                           size_t workspace_bytes, void* stream) {
  if (int rc = check_embedding("esa_embedding_backward", dtype, id_bytes, n_tokens, vocab, dim, ids,
                               scale))
    return rc;
  if ((n_tokens > 0 && (!dy || !aligned16(dy))) || !dweight || !aligned16(dweight))
    return fail(ESA_ERR_INVALID, "esa_embedding_backward: null or misaligned pointer");
  const size_t need = esa_embedding_backward_workspace_size(n_tokens, vocab, dim);
  if (need && (!workspace || workspace_bytes < need))
    return fail(ESA_ERR_WORKSPACE, "esa_embedding_backward: workspace of %zu bytes given, %zu needed",
                workspace_bytes, need);
  if (need && reinterpret_cast<uintptr_t>(workspace) % 256)
    return fail(ESA_ERR_INVALID, "esa_embedding_backward: workspace must be 256-byte aligned");
  int* err = nullptr;
  if (int rc = device_error_word(&err)) return rc;
  const em::Ids src{ids, id_bytes == 8};
  return by_dtype(dtype, [&](auto tag) {
    return embedding_grad<decltype(tag)>(n_tokens, vocab, dim, src, dy, scale,
                                         padding_idx < 0 ? -1 : padding_idx, dweight,
                                         static_cast<char*>(workspace), err, (cudaStream_t)stream);
  });
}

int esa_qk_norm_rope_forward(int32_t dtype, int32_t batch, int64_t seq_len, int32_t head_dim,
                             esa_tensor_t q, int32_t num_q_heads, esa_tensor_t k,
                             int32_t num_k_heads, const void* q_weight, const void* k_weight,
                             float eps, const int64_t* positions, int64_t positions_stride_b,
                             const float* inv_freq, esa_tensor_t q_out, esa_tensor_t k_out,
                             void* stream) {
  if (int rc = check_qk("esa_qk_norm_rope_forward", dtype, batch, seq_len, head_dim, num_q_heads,
                        num_k_heads, positions_stride_b, eps))
    return rc;
  if (batch == 0 || seq_len == 0 || num_q_heads + num_k_heads == 0) return ESA_OK;
  if (!inv_freq) return fail(ESA_ERR_INVALID, "esa_qk_norm_rope_forward: null inv_freq");
  return by_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    qk::Params<T> p;
    if (int rc = set_heads(p.q, "q", q, nullptr, q_out, q_weight, num_q_heads)) return rc;
    if (int rc = set_heads(p.k, "k", k, nullptr, k_out, k_weight, num_k_heads)) return rc;
    p.L = seq_len;
    p.tokens = (int64_t)batch * seq_len;
    p.pos = positions;
    p.pos_sb = positions_stride_b;
    p.inv_freq = inv_freq;
    p.eps = eps;
    const int tpr = head_dim / (2 * esa::Vec<T>::kElems);
    set_tasks(p, 32 / tpr);
    const int64_t ctas = p.nt > 1 ? ceil_div(p.tokens, (int64_t)p.nt * qk::kWarps)
                                  : ceil_div(p.tokens * p.tasks, qk::kWarps);
    if (ctas > INT32_MAX)
      return fail(ESA_ERR_UNSUPPORTED, "esa_qk_norm_rope_forward: too many positions");
    return by_threads_per_row<1>(tpr, [&](auto t) {
      constexpr int TPR = decltype(t)::value;
      cudaStream_t s = (cudaStream_t)stream;
      if (p.nt > 1)
        qk::fwd_few_kernel<T, TPR><<<(unsigned)ctas, qk::kThreads, 0, s>>>(p);
      else
        qk::fwd_kernel<T, TPR><<<(unsigned)ctas, qk::kThreads, 0, s>>>(p);
      return check_launch("esa_qk_norm_rope_forward");
    });
  });
}

size_t esa_qk_norm_rope_backward_workspace_size(int32_t batch, int64_t seq_len, int32_t num_q_heads,
                                                int32_t num_k_heads, int32_t head_dim) {
  if (batch <= 0 || seq_len <= 0 || num_q_heads < 0 || num_k_heads < 0 || head_dim <= 0) return 0;
  return (size_t)qk_bwd_ctas((int64_t)batch * seq_len, num_q_heads, num_k_heads) * head_dim *
         sizeof(float);
}

int esa_qk_norm_rope_backward(int32_t dtype, int32_t batch, int64_t seq_len, int32_t head_dim,
                              esa_tensor_t q, int32_t num_q_heads, esa_tensor_t k,
                              int32_t num_k_heads, const void* q_weight, const void* k_weight,
                              float eps, const int64_t* positions, int64_t positions_stride_b,
                              const float* inv_freq, esa_tensor_t dq_out, esa_tensor_t dk_out,
                              esa_tensor_t dq, esa_tensor_t dk, void* dq_weight, void* dk_weight,
                              void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_qk("esa_qk_norm_rope_backward", dtype, batch, seq_len, head_dim, num_q_heads,
                        num_k_heads, positions_stride_b, eps))
    return rc;
  if ((num_q_heads > 0 && !dq_weight) || (num_k_heads > 0 && !dk_weight))
    return fail(ESA_ERR_INVALID, "esa_qk_norm_rope_backward: null weight gradient");
  cudaStream_t s = (cudaStream_t)stream;
  const bool no_tokens = batch == 0 || seq_len == 0;   // sums over no rows are zero
  const size_t weight_bytes = (size_t)head_dim * elem_size(dtype);
  if (dq_weight && (no_tokens || num_q_heads == 0)) cudaMemsetAsync(dq_weight, 0, weight_bytes, s);
  if (dk_weight && (no_tokens || num_k_heads == 0)) cudaMemsetAsync(dk_weight, 0, weight_bytes, s);
  if (no_tokens || num_q_heads + num_k_heads == 0) return check_launch("esa_qk_norm_rope_backward");
  if (!inv_freq) return fail(ESA_ERR_INVALID, "esa_qk_norm_rope_backward: null inv_freq");
  const size_t need = esa_qk_norm_rope_backward_workspace_size(batch, seq_len, num_q_heads,
                                                               num_k_heads, head_dim);
  if (!workspace || workspace_bytes < need)
    return fail(ESA_ERR_WORKSPACE,
                "esa_qk_norm_rope_backward: workspace of %zu bytes given, %zu needed",
                workspace_bytes, need);
  if (!aligned16(workspace))
    return fail(ESA_ERR_INVALID, "esa_qk_norm_rope_backward: workspace must be 16-byte aligned");
  return by_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    qk::Params<T> p;
    if (int rc = set_heads(p.q, "q", q, &dq_out, dq, q_weight, num_q_heads)) return rc;
    if (int rc = set_heads(p.k, "k", k, &dk_out, dk, k_weight, num_k_heads)) return rc;
    p.L = seq_len;
    p.tokens = (int64_t)batch * seq_len;
    p.pos = positions;
    p.pos_sb = positions_stride_b;
    p.inv_freq = inv_freq;
    p.eps = eps;
    const int tpr = head_dim / 8;   // four elements of each half per thread
    set_tasks(p, 32 / tpr);
    const int ctas = qk_bwd_ctas(p.tokens, num_q_heads, num_k_heads);
    const int q_ctas = qk_q_ctas(p, ctas);
    float* part = static_cast<float*>(workspace);
    return by_threads_per_row<esa::Vec<T>::kElems / 4>(tpr, [&](auto t) {
      qk::bwd_kernel<T, decltype(t)::value><<<ctas, qk::kThreads, 0, s>>>(p, q_ctas, part);
      if (int rc = check_launch("esa_qk_norm_rope_backward")) return rc;
      // block row 0: query weights, 1: key weights
      const int first = num_q_heads > 0 ? 0 : 1, sides = (num_q_heads > 0) + (num_k_heads > 0);
      return launch_after("esa_qk_norm_rope_backward (weight sums)", qk::sum_kernel<T>,
                          dim3((unsigned)ceil_div(head_dim, 32), sides), dim3(qk::kSumWarps * 32),
                          s, head_dim, q_ctas, ctas, first, part, static_cast<T*>(dq_weight),
                          static_cast<T*>(dk_weight));
    });
  });
}

int esa_quantize_rows(int32_t dtype, int32_t format, int64_t n_rows, int32_t dim, const void* x,
                      void* codes, float* scales, void* stream) {
  if (int rc = check_pack("esa_quantize_rows", dtype, format, n_rows, dim)) return rc;
  if (n_rows == 0) return ESA_OK;
  if (!x || !codes || !scales || !aligned16(x) || !aligned16(codes) || !aligned16(scales))
    return fail(ESA_ERR_INVALID, "esa_quantize_rows: null or misaligned pointer");
  return by_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    return by_format(format, [&](auto f) {
      p8::quantize_kernel<T, decltype(f)::value>
          <<<part_grid(n_rows, dim, esa::Vec<T>::kElems, p8::kRowUnits), p8::kThreads, 0, (cudaStream_t)stream>>>(
              n_rows, dim, static_cast<const T*>(x), static_cast<uint8_t*>(codes), scales);
      return check_launch("esa_quantize_rows");
    });
  });
}

int esa_dequantize_rows(int32_t dtype, int32_t format, int64_t n_rows, int32_t dim,
                        const void* codes, const float* scales, void* x, void* stream) {
  if (int rc = check_pack("esa_dequantize_rows", dtype, format, n_rows, dim)) return rc;
  if (n_rows == 0) return ESA_OK;
  if (!x || !codes || !scales || !aligned16(x) || !aligned16(codes) || !aligned16(scales))
    return fail(ESA_ERR_INVALID, "esa_dequantize_rows: null or misaligned pointer");
  return by_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    return by_format(format, [&](auto f) {
      p8::dequantize_kernel<T, decltype(f)::value>
          <<<part_grid(n_rows, dim, esa::Vec<T>::kElems, p8::kRowUnits), p8::kThreads, 0, (cudaStream_t)stream>>>(
              n_rows, dim, static_cast<const uint8_t*>(codes), scales, static_cast<T*>(x));
      return check_launch("esa_dequantize_rows");
    });
  });
}

int esa_rmsnorm_pack_forward(int32_t dtype, int32_t format, int64_t n_rows, int32_t dim,
                             const void* x, const void* residual, void* h_out, const void* weight,
                             float eps, void* y, float* rstd, void* codes, float* scales,
                             void* stream) {
  if (int rc = check_pack("esa_rmsnorm_pack_forward", dtype, format, n_rows, dim)) return rc;
  if (int rc = check_norm_rows("esa_rmsnorm_pack_forward", dtype, n_rows, dim, eps)) return rc;
  if (n_rows == 0) return ESA_OK;
  if (!x || !weight || !y || !rstd || !codes || !scales || (residual && !h_out) || !aligned16(x) ||
      !aligned16(weight) || !aligned16(y) || !aligned16(codes) || !aligned16(scales) ||
      !aligned16(residual) || !aligned16(h_out))
    return fail(ESA_ERR_INVALID, "esa_rmsnorm_pack_forward: null or misaligned pointer");
  return by_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    return by_format(format, [&](auto f) {
      return by_row_shape(dim / esa::Vec<T>::kElems, [&](auto nv, auto nw) {
        constexpr int W = decltype(nw)::value;
        p8::norm_pack_kernel<T, decltype(f)::value, decltype(nv)::value, W>
            <<<(unsigned)ceil_div(n_rows, p8::kNormRows<W>), p8::kNormThreads<W>, 0,
               (cudaStream_t)stream>>>(n_rows, dim, static_cast<const T*>(x),
                                       static_cast<const T*>(residual), static_cast<T*>(h_out),
                                       static_cast<const T*>(weight), eps, static_cast<T*>(y), rstd,
                                       static_cast<uint8_t*>(codes), scales);
        return check_launch("esa_rmsnorm_pack_forward");
      });
    });
  });
}

int esa_rmsnorm_unpack_forward(int32_t dtype, int32_t format, int64_t n_rows, int32_t dim,
                               const void* codes, const float* scales, const void* weight,
                               float eps, void* h, void* y, float* rstd, void* stream) {
  if (int rc = check_pack("esa_rmsnorm_unpack_forward", dtype, format, n_rows, dim)) return rc;
  if (int rc = check_norm_rows("esa_rmsnorm_unpack_forward", dtype, n_rows, dim, eps)) return rc;
  if (n_rows == 0) return ESA_OK;
  if (!codes || !scales || !weight || !h || !y || !rstd || !aligned16(codes) ||
      !aligned16(scales) || !aligned16(weight) || !aligned16(h) || !aligned16(y))
    return fail(ESA_ERR_INVALID, "esa_rmsnorm_unpack_forward: null or misaligned pointer");
  return by_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    return by_format(format, [&](auto f) {
      return by_row_shape(dim / esa::Vec<T>::kElems, [&](auto nv, auto nw) {
        constexpr int W = decltype(nw)::value;
        p8::unpack_norm_kernel<T, decltype(f)::value, decltype(nv)::value, W>
            <<<(unsigned)ceil_div(n_rows, p8::kNormRows<W>), p8::kNormThreads<W>, 0,
               (cudaStream_t)stream>>>(n_rows, dim, static_cast<const uint8_t*>(codes), scales,
                                       static_cast<T*>(h), static_cast<const T*>(weight), eps,
                                       static_cast<T*>(y), rstd);
        return check_launch("esa_rmsnorm_unpack_forward");
      });
    });
  });
}

int esa_swiglu_pack_forward(int32_t dtype, int32_t format, int64_t n_rows, int32_t ffn,
                            const void* gate_up, void* out, void* codes, float* scales,
                            void* stream) {
  if (int rc = check_pack("esa_swiglu_pack_forward", dtype, format, n_rows, ffn)) return rc;
  if (n_rows == 0) return ESA_OK;
  if (!gate_up || !out || !codes || !scales || !aligned16(gate_up) || !aligned16(out) ||
      !aligned16(codes) || !aligned16(scales))
    return fail(ESA_ERR_INVALID, "esa_swiglu_pack_forward: null or misaligned pointer");
  return by_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    return by_format(format, [&](auto f) {
      p8::swiglu_pack_kernel<T, decltype(f)::value>
          <<<part_grid(n_rows, ffn, esa::Vec<T>::kElems, p8::kSwigluFwdUnits), p8::kThreads, 0, (cudaStream_t)stream>>>(
              n_rows, ffn, static_cast<const T*>(gate_up), static_cast<T*>(out),
              static_cast<uint8_t*>(codes), scales);
      return check_launch("esa_swiglu_pack_forward");
    });
  });
}

int esa_swiglu_unpack_backward(int32_t dtype, int32_t format, int64_t n_rows, int32_t ffn,
                               const void* codes, const float* scales, const void* dout,
                               void* dgate_up, void* out_recomputed, void* stream) {
  if (int rc = check_pack("esa_swiglu_unpack_backward", dtype, format, n_rows, ffn)) return rc;
  if (n_rows == 0) return ESA_OK;
  if (!codes || !scales || !dout || !dgate_up || !aligned16(codes) || !aligned16(scales) ||
      !aligned16(dout) || !aligned16(dgate_up) || !aligned16(out_recomputed))
    return fail(ESA_ERR_INVALID, "esa_swiglu_unpack_backward: null or misaligned pointer");
  return by_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    return by_format(format, [&](auto f) {
      p8::swiglu_unpack_bwd_kernel<T, decltype(f)::value>
          <<<part_grid(n_rows, ffn, esa::Vec<T>::kElems, p8::kSwigluBwdUnits), p8::kThreads, 0, (cudaStream_t)stream>>>(
              n_rows, ffn, static_cast<const uint8_t*>(codes), scales, static_cast<const T*>(dout),
              static_cast<T*>(dgate_up), static_cast<T*>(out_recomputed));
      return check_launch("esa_swiglu_unpack_backward");
    });
  });
}

}  // extern "C"
