// extern "C" entry points of include/esa_layer.h: log probabilities of tokens and
// their gradient, products with weights in 4 bits, the key / value cache in 4 bits
// and the attention over it.
#include <algorithm>
#include <atomic>
#include <cmath>

#include "esa_layer.h"
#include "esa_cache4.cuh"
#include "esa_host.h"
#include "esa_score.cuh"
#include "esa_weight4.cuh"

namespace {

using namespace esa::host;

constexpr int kSms = 148;
constexpr int64_t kMaxGrid = (int64_t(1) << 31) - 1;

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

bool known_dtype(int32_t d) { return d == ESA_DTYPE_F32 || d == ESA_DTYPE_BF16 || d == ESA_DTYPE_F16; }

// Launches `kernel` with clusters of `ctas` neighbouring CTAs; its CTAs may be placed
// while the kernel before it still runs (see launch_after).
template <typename Q>
int launch_clusters(const char* what, void (*kernel)(const Q), dim3 grid, dim3 block, int ctas,
                    cudaStream_t s, const Q& params, size_t shared = 0) {
  cudaLaunchConfig_t c = {};
  c.gridDim = grid;
  c.blockDim = block;
  c.dynamicSmemBytes = shared;
  c.stream = s;
  cudaLaunchAttribute a[2];
  a[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  a[0].val.programmaticStreamSerializationAllowed = 1;
  a[1].id = cudaLaunchAttributeClusterDimension;
  a[1].val.clusterDim.x = ctas;
  a[1].val.clusterDim.y = 1;
  a[1].val.clusterDim.z = 1;
  c.attrs = a;
  c.numAttrs = ctas > 1 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&c, kernel, params);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(ESA_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
  }
  return ESA_OK;
}

// ---------------------------------------------------------------------------
// Log probabilities.
// ---------------------------------------------------------------------------
namespace sc = esa::score;

int check_score(const char* what, int32_t dtype, int32_t id_bytes, int64_t n_rows, int64_t vocab,
                int64_t row_stride, const void* logits, const void* tokens) {
  if (!known_dtype(dtype)) return fail(ESA_ERR_INVALID, "%s: unknown dtype %d", what, dtype);
  if (id_bytes != 4 && id_bytes != 8)
    return fail(ESA_ERR_INVALID, "%s: id_bytes %d (4 or 8)", what, id_bytes);
  if (n_rows < 0 || vocab < 1) return fail(ESA_ERR_INVALID, "%s: bad shape", what);
  if (row_stride < vocab && n_rows > 1)
    return fail(ESA_ERR_INVALID, "%s: row stride %lld below the vocabulary", what, (long long)row_stride);
  if (vocab > kMaxGrid || n_rows > kMaxGrid / 8)
    return fail(ESA_ERR_UNSUPPORTED, "%s: 2^31 elements in a row, or 2^28 rows", what);
  if (n_rows > 0 && (!logits || reinterpret_cast<uintptr_t>(logits) % elem_size(dtype) || !tokens ||
                     reinterpret_cast<uintptr_t>(tokens) % id_bytes))
    return fail(ESA_ERR_INVALID, "%s: null or misaligned logits or tokens", what);
  return ESA_OK;
}

// ---------------------------------------------------------------------------
// Weights in 4 bits.
// ---------------------------------------------------------------------------
namespace w4 = esa::w4;

int check_weight4(const char* what, int32_t dtype, int64_t n, int64_t k, int32_t group,
                  const void* codes, const void* scales) {
  if (!known_dtype(dtype)) return fail(ESA_ERR_INVALID, "%s: unknown dtype %d", what, dtype);
  if (n < 1 || k < 1) return fail(ESA_ERR_INVALID, "%s: bad shape", what);
  if (n > (int64_t(1) << 20) || k > (int64_t(1) << 20))
    return fail(ESA_ERR_UNSUPPORTED, "%s: more than 2^20 rows or inputs", what);
  if ((k * elem_size(dtype)) % 16)
    return fail(ESA_ERR_INVALID, "%s: k * element size must be a multiple of 16 bytes", what);
  if (group != 32 && group != 64 && group != 128)
    return fail(ESA_ERR_INVALID, "%s: group %d (32, 64 or 128)", what, group);
  if (!codes || !scales || !aligned16(codes) || !aligned16(scales))
    return fail(ESA_ERR_INVALID, "%s: null or misaligned codes or scales", what);
  return ESA_OK;
}

w4::Packed packed(int64_t n, int64_t k, int32_t group, const void* codes, const void* scales) {
  w4::Packed p;
  p.codes = static_cast<uint8_t*>(const_cast<void*>(codes));
  p.scales = static_cast<__nv_bfloat16*>(const_cast<void*>(scales));
  p.N = (int)n;
  p.K = (int)k;
  p.group = group;
  p.tiles = (int)ceil_div(n, w4::kTileRows);
  p.chunks = (int)ceil_div(k, w4::kTileK);
  p.groups = p.chunks * (w4::kTileK / group);
  return p;
}

// Allows `kernel` its shared memory on the current device, once per device (the call
// takes a good part of a launch's time on the host).  `done` is the kernel's own.
template <typename K>
int reserve_shared(const char* what, K* kernel, int bytes, std::atomic<uint64_t>& done) {
  if (bytes <= 48 * 1024) return ESA_OK;
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) device = 64;
  const uint64_t bit = device < 64 ? uint64_t(1) << device : 0;
  if (done.load(std::memory_order_relaxed) & bit) return ESA_OK;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) {
    cudaGetLastError();
    return fail(ESA_ERR_CUDA, "%s: cannot reserve %d bytes of shared memory", what, bytes);
  }
  done.fetch_or(bit, std::memory_order_relaxed);
  return ESA_OK;
}

// Up to 8 columns: as many warps on a tile of rows as leave all of them resident
// (some 24 per SM), with two tiles of K per warp at least.
template <typename T, int G>
int linear_vector(const w4::LinearParams<T>& p, cudaStream_t s) {
  auto go = [&](auto wk) {
    constexpr int WK = decltype(wk)::value;
    constexpr int kShared = WK * w4::kDepth * w4::Tile<G>::kBytes;
    auto* kernel = w4::vector_kernel<T, G, WK>;
    static std::atomic<uint64_t> done{0};
    if (int rc = reserve_shared("esa_linear4", kernel, kShared, done)) return rc;
    return launch_clusters("esa_linear4", kernel, dim3((unsigned)p.tiles), dim3(WK * 32), 1, s, p,
                           kShared);
  };
  int wk = 2;
  while (wk < 16 && p.tiles * wk * 2 <= kSms * 32 && p.chunks >= wk * 4) wk *= 2;
  switch (wk) {
    case 2: return go(std::integral_constant<int, 2>{});
    case 4: return go(std::integral_constant<int, 4>{});
    case 8: return go(std::integral_constant<int, 8>{});
    default: return go(std::integral_constant<int, 16>{});
  }
}

// More columns: K is split over a cluster until there are up to three CTAs per SM
// (two are resident: 32 x 4096 x 12288 takes 18 us with 384 CTAs, 21 with 192), with
// two stages at least.
template <typename T, int G, int NT>
int linear_rows(const w4::LinearParams<T>& p, cudaStream_t s) {
  using S = w4::Shape<T, G, NT>;
  const int64_t row_ctas = ceil_div(p.tiles, w4::kWarps), col_ctas = ceil_div(p.M, S::kTokens);
  if (col_ctas > 65535) return fail(ESA_ERR_UNSUPPORTED, "esa_linear4: too many rows");
  int ctas = 1;
  while (ctas < 8 && row_ctas * col_ctas * ctas * 2 <= kSms * 3 && p.chunks >= ctas * 2 * 2 * S::kStage)
    ctas *= 2;
  auto* kernel = w4::rows_kernel<T, G, NT>;
  static std::atomic<uint64_t> done{0};
  if (int rc = reserve_shared("esa_linear4", kernel, S::kShared, done)) return rc;
  return launch_clusters("esa_linear4", kernel, dim3((unsigned)(row_ctas * ctas), (unsigned)col_ctas),
                         dim3(w4::kWarps * 32), ctas, s, p, S::kShared);
}

template <typename T, int G>
int linear(const w4::LinearParams<T>& p, cudaStream_t s) {
  const int64_t cols = (int64_t)p.M * w4::Operand<T>::kParts;
  // float32 rows are cut in three parts, which a CTA of 128 weight rows does once where
  // eight of 16 do it each (2 x 4096 x 4096: 12 -> 6 us)
  if constexpr (w4::Operand<T>::kParts == 1)
    if (cols <= 8) return linear_vector<T, G>(p, s);
  if (cols <= 16) return linear_rows<T, G, 2>(p, s);
  if (cols <= 32) return linear_rows<T, G, 4>(p, s);
  return linear_rows<T, G, 8>(p, s);
}

// ---------------------------------------------------------------------------
// Cache in 4 bits.
// ---------------------------------------------------------------------------
namespace c4 = esa::cache4;

int check_cache(const char* what, int32_t dtype, const esa_cache4_t* c, int64_t rows,
                int64_t start0, const int64_t* start, const int64_t* counts) {
  if (!known_dtype(dtype)) return fail(ESA_ERR_INVALID, "%s: unknown dtype %d", what, dtype);
  if (!c) return fail(ESA_ERR_INVALID, "%s: null cache", what);
  if (c->batch < 0 || c->num_kv_heads < 1 || c->max_len < 1 || rows < 0)
    return fail(ESA_ERR_INVALID, "%s: bad shape", what);
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
    return fail(ESA_ERR_UNSUPPORTED, "%s: head_dim %d (64, 128 or 256)", what, c->head_dim);
  if (c->max_len > esa::kMaxPosition)
    return fail(ESA_ERR_UNSUPPORTED, "%s: max_len above 2^24", what);
  if (rows > esa::kMaxPosition) return fail(ESA_ERR_INVALID, "%s: more rows than positions", what);
  if (!start && start0 < 0) return fail(ESA_ERR_INVALID, "%s: negative start", what);
  if (reinterpret_cast<uintptr_t>(start) % 8 || reinterpret_cast<uintptr_t>(counts) % 8)
    return fail(ESA_ERR_INVALID, "%s: misaligned start or counts", what);
  if (c->batch == 0) return ESA_OK;            // no memory: there is nothing to read or write
  if (!c->codes || !c->scales || !aligned16(c->codes) || !aligned16(c->scales))
    return fail(ESA_ERR_INVALID, "%s: null or misaligned codes or scales", what);
  return ESA_OK;
}

c4::Cache cache_of(const esa_cache4_t* c) {
  c4::Cache r;
  r.codes = static_cast<uint8_t*>(c->codes);
  r.scales = static_cast<__nv_bfloat16*>(c->scales);
  r.B = c->batch;
  r.Hkv = c->num_kv_heads;
  r.S = c->max_len;
  return r;
}

c4::Heads heads_of(const esa_tensor_t& t) { return {t.data, t.stride_b, t.stride_h, t.stride_s}; }

template <typename F>
int by_head_dim(int32_t d, F&& f) {
  switch (d) {
    case 64: return f(std::integral_constant<int, 64>{});
    case 128: return f(std::integral_constant<int, 128>{});
    default: return f(std::integral_constant<int, 256>{});
  }
}

int cache_rows(const char* what, bool write, int32_t dtype, const esa_cache4_t* cache,
               int64_t seq_len, esa_tensor_t k, esa_tensor_t v, const int64_t* start,
               int64_t start0, const int64_t* counts, void* stream) {
  if (int rc = check_cache(what, dtype, cache, seq_len, start0, start, counts)) return rc;
  if (seq_len == 0 || cache->batch == 0) return ESA_OK;
  if (int rc = check_tensor("k", k, elem_size(dtype))) return rc;
  if (int rc = check_tensor("v", v, elem_size(dtype))) return rc;
  const int64_t rows = seq_len * cache->num_kv_heads;
  if (rows > kMaxGrid || cache->batch > 65535)
    return fail(ESA_ERR_UNSUPPORTED, "%s: more than 2^31 rows of a sequence, or 65535 sequences", what);
  int* err = nullptr;
  if (int rc = device_error_word(&err)) return rc;
  return by_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    c4::RowParams<T> p;
    p.c = cache_of(cache);
    p.span = {start, counts, start0, seq_len};
    p.k = heads_of(k);
    p.v = heads_of(v);
    p.rows = (unsigned)rows;
    p.err = err;
    return by_head_dim(cache->head_dim, [&](auto d) {
      constexpr int D = decltype(d)::value;
      const dim3 grid((unsigned)ceil_div(rows, c4::Unit<D>::kRows * c4::kRowsPerThread),
                      (unsigned)cache->batch);
      if (write)
        c4::write_kernel<T, D><<<grid, c4::kRowThreads, 0, (cudaStream_t)stream>>>(p);
      else
        c4::read_kernel<T, D><<<grid, c4::kRowThreads, 0, (cudaStream_t)stream>>>(p);
      return check_launch(what);
    });
  });
}

}  // namespace

extern "C" {

int esa_token_logprobs_forward(int32_t dtype, int32_t id_bytes, int64_t n_rows, int64_t vocab,
                               int64_t row_stride, const void* logits, const void* tokens,
                               int32_t top_k, float* logprobs, float* entropy, float* stats,
                               int64_t* top_ids, float* top_logprobs, void* stream) {
  const char* what = "esa_token_logprobs_forward";
  if (int rc = check_score(what, dtype, id_bytes, n_rows, vocab, row_stride, logits, tokens)) return rc;
  if (top_k < 0 || top_k > sc::kMaxTop || top_k > vocab)
    return fail(ESA_ERR_INVALID, "%s: top_k %d outside [0, min(%d, vocab)]", what, top_k, sc::kMaxTop);
  if (n_rows == 0) return ESA_OK;
  if (!logprobs || !entropy || !stats || reinterpret_cast<uintptr_t>(stats) % 8 ||
      (top_k > 0 && (!top_ids || !top_logprobs)))
    return fail(ESA_ERR_INVALID, "%s: null or misaligned output", what);
  int* err = nullptr;
  if (int rc = device_error_word(&err)) return rc;
  return by_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    sc::FwdParams<T> p;
    p.logits = static_cast<const T*>(logits);
    p.stride = row_stride;
    p.V = vocab;
    p.tokens = tokens;
    p.id_bytes = id_bytes;
    p.top = top_k;
    p.logprobs = logprobs;
    p.entropy = entropy;
    p.stats = reinterpret_cast<float2*>(stats);
    p.top_ids = top_ids;
    p.top_logprobs = top_logprobs;
    p.err = err;
    const int64_t vecs = vocab / esa::Vec<T>::kElems;
    auto go = [&](auto nw) {
      constexpr int NW = decltype(nw)::value;
      // few rows: a row over up to 8 CTAs, with a vector per thread at least, until there
      // is a CTA per SM (333 x 50021 float32, beyond that, takes 20 us, split in four 24;
      // in two was not tried)
      int ctas = 1;
      while (ctas < 8 && n_rows * ctas < kSms && vecs >= (int64_t)ctas * 2 * NW * 32) ctas *= 2;
      const dim3 grid((unsigned)(n_rows * ctas)), block(NW * 32);
      if (top_k > 0)
        return launch_clusters(what, sc::fwd_kernel<T, NW, true>, grid, block, ctas,
                               (cudaStream_t)stream, p);
      return launch_clusters(what, sc::fwd_kernel<T, NW, false>, grid, block, ctas,
                             (cudaStream_t)stream, p);
    };
    if (vecs <= 512) return go(std::integral_constant<int, 2>{});
    return go(std::integral_constant<int, 8>{});
  });
}

int esa_token_logprobs_backward(int32_t dtype, int32_t id_bytes, int64_t n_rows, int64_t vocab,
                                int64_t row_stride, const void* logits, const void* tokens,
                                const float* stats, const float* entropy, const float* dlogprobs,
                                const float* dentropy, int64_t dlogits_stride, void* dlogits,
                                void* stream) {
  const char* what = "esa_token_logprobs_backward";
  if (int rc = check_score(what, dtype, id_bytes, n_rows, vocab, row_stride, logits, tokens)) return rc;
  if (n_rows == 0) return ESA_OK;
  if (dlogits_stride < vocab && n_rows > 1)
    return fail(ESA_ERR_INVALID, "%s: gradient row stride below the vocabulary", what);
  if (!stats || reinterpret_cast<uintptr_t>(stats) % 8 || !entropy || !dlogits ||
      reinterpret_cast<uintptr_t>(dlogits) % elem_size(dtype))
    return fail(ESA_ERR_INVALID, "%s: null or misaligned pointer", what);
  if (dlogits == logits && n_rows > 1 && dlogits_stride != row_stride)
    return fail(ESA_ERR_INVALID, "%s: in place with another row stride", what);
  int* err = nullptr;
  if (int rc = device_error_word(&err)) return rc;
  return by_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    sc::BwdParams<T> p;
    p.logits = static_cast<const T*>(logits);
    p.dlogits = static_cast<T*>(dlogits);
    p.stride = row_stride;
    p.dstride = dlogits_stride;
    p.V = vocab;
    p.tokens = tokens;
    p.id_bytes = id_bytes;
    p.stats = reinterpret_cast<const float2*>(stats);
    p.entropy = entropy;
    p.dlogprobs = dlogprobs;
    p.dentropy = dentropy;
    p.err = err;
    const int64_t parts = std::max<int64_t>(1, ceil_div(vocab / esa::Vec<T>::kElems, sc::kBwdVecs));
    if (n_rows * parts > kMaxGrid) return fail(ESA_ERR_UNSUPPORTED, "%s: too many elements", what);
    p.parts = (unsigned)parts;
    sc::bwd_kernel<T><<<(unsigned)(n_rows * parts), sc::kBwdThreads, 0, (cudaStream_t)stream>>>(p);
    return check_launch(what);
  });
}

size_t esa_weight4_codes_size(int64_t n, int64_t k) {
  if (n < 1 || k < 1) return 0;
  return (size_t)ceil_div(n, w4::kTileRows) * ceil_div(k, w4::kTileK) * w4::kTileBytes;
}

int esa_quantize_weight4(int32_t dtype, int64_t n, int64_t k, int32_t group, const void* weight,
                         void* codes, void* scales, void* stream) {
  const char* what = "esa_quantize_weight4";
  if (int rc = check_weight4(what, dtype, n, k, group, codes, scales)) return rc;
  if (!weight || !aligned16(weight)) return fail(ESA_ERR_INVALID, "%s: null or misaligned weight", what);
  const w4::Packed p = packed(n, k, group, codes, scales);
  const dim3 grid((unsigned)p.chunks * (unsigned)p.tiles);       // up to 2^29
  return by_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    w4::quantize_kernel<T><<<grid, w4::kPackThreads, 0, (cudaStream_t)stream>>>(
        p, static_cast<const T*>(weight));
    return check_launch(what);
  });
}

int esa_dequantize_weight4(int32_t dtype, int64_t n, int64_t k, int32_t group, const void* codes,
                           const void* scales, void* weight, void* stream) {
  const char* what = "esa_dequantize_weight4";
  if (int rc = check_weight4(what, dtype, n, k, group, codes, scales)) return rc;
  if (!weight || !aligned16(weight)) return fail(ESA_ERR_INVALID, "%s: null or misaligned weight", what);
  const w4::Packed p = packed(n, k, group, codes, scales);
  const dim3 grid((unsigned)p.chunks * (unsigned)p.tiles);       // up to 2^29
  return by_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    w4::dequantize_kernel<T><<<grid, w4::kPackThreads, 0, (cudaStream_t)stream>>>(
        p, static_cast<T*>(weight));
    return check_launch(what);
  });
}

int esa_linear4(int32_t dtype, int64_t n_rows, int64_t n, int64_t k, int32_t group, const void* x,
                const void* codes, const void* scales, void* y, void* stream) {
  const char* what = "esa_linear4";
  if (int rc = check_weight4(what, dtype, n, k, group, codes, scales)) return rc;
  if (n_rows < 0 || n_rows > (int64_t(1) << 20))
    return fail(ESA_ERR_INVALID, "%s: n_rows %lld", what, (long long)n_rows);
  if (n_rows == 0) return ESA_OK;
  if (!x || !y || !aligned16(x) || !aligned16(y))
    return fail(ESA_ERR_INVALID, "%s: null or misaligned x or y", what);
  const w4::Packed w = packed(n, k, group, codes, scales);
  return by_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    w4::LinearParams<T> p;
    p.x = static_cast<const T*>(x);
    p.y = static_cast<T*>(y);
    p.codes = w.codes;
    p.scales = w.scales;
    p.M = (int)n_rows;
    p.N = w.N;
    p.K = w.K;
    p.tiles = w.tiles;
    p.chunks = w.chunks;
    cudaStream_t s = (cudaStream_t)stream;
    switch (group) {
      case 32: return linear<T, 32>(p, s);
      case 64: return linear<T, 64>(p, s);
      default: return linear<T, 128>(p, s);
    }
  });
}

int esa_cache4_write(int32_t dtype, const esa_cache4_t* cache, int64_t seq_len, esa_tensor_t k,
                     esa_tensor_t v, const int64_t* start, int64_t start0, const int64_t* counts,
                     void* stream) {
  return cache_rows("esa_cache4_write", true, dtype, cache, seq_len, k, v, start, start0, counts,
                    stream);
}

int esa_cache4_read(int32_t dtype, const esa_cache4_t* cache, int64_t seq_len, esa_tensor_t k,
                    esa_tensor_t v, const int64_t* start, int64_t start0, void* stream) {
  return cache_rows("esa_cache4_read", false, dtype, cache, seq_len, k, v, start, start0, nullptr,
                    stream);
}

int esa_cache4_forward(int32_t dtype, const esa_cache4_t* cache, int32_t num_heads, int64_t q_len,
                       int32_t attn_length, int32_t layer_idx, int32_t num_hidden_layers,
                       int32_t pattern_heads, int32_t head_offset, float scale, esa_tensor_t q,
                       const int64_t* start, int64_t start0, const int64_t* counts, esa_tensor_t o,
                       float* lse, void* stream) {
  const char* what = "esa_cache4_forward";
  if (int rc = check_cache(what, dtype, cache, q_len, start0, start, counts)) return rc;
  if (num_heads < 1 || num_heads % cache->num_kv_heads)
    return fail(ESA_ERR_INVALID, "%s: num_heads (%d) must be divisible by num_kv_heads (%d)", what,
                num_heads, cache->num_kv_heads);
  if (attn_length < 1 || attn_length > esa::kMaxAttnLength)
    return fail(ESA_ERR_UNSUPPORTED, "%s: attention_length %d outside [1, %d]", what, attn_length,
                esa::kMaxAttnLength);
  if (num_hidden_layers < 1 || layer_idx < 0 || layer_idx >= num_hidden_layers)
    return fail(ESA_ERR_INVALID, "%s: layer %d of %d", what, layer_idx, num_hidden_layers);
  const int32_t heads = pattern_heads > 0 ? pattern_heads : num_heads;
  if (pattern_heads < 0 || head_offset < 0 || (int64_t)head_offset + num_heads > heads || heads > 65535)
    return fail(ESA_ERR_INVALID, "%s: head_offset %d + num_heads %d must be <= pattern_heads %d (<= 65535)",
                what, head_offset, num_heads, heads);
  if (!std::isfinite(scale)) return fail(ESA_ERR_INVALID, "%s: scale must be finite", what);
  if (q_len == 0 || cache->batch == 0) return ESA_OK;
  if (int rc = check_tensor("q", q, elem_size(dtype))) return rc;
  if (int rc = check_tensor("o", o, elem_size(dtype))) return rc;
  if (!lse) return fail(ESA_ERR_INVALID, "%s: null lse", what);
  const int64_t pairs = (int64_t)cache->batch * num_heads * q_len;
  const int64_t rows = num_heads / cache->num_kv_heads * q_len;
  const int64_t kv = (int64_t)cache->batch * cache->num_kv_heads;
  if (rows > kMaxGrid || kv > 65535)
    return fail(ESA_ERR_UNSUPPORTED, "%s: more than 2^31 rows per K/V head, or 65535 K/V heads", what);
  int* err = nullptr;
  if (int rc = device_error_word(&err)) return rc;
  return by_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    c4::AttendParams<T> p;
    p.c = cache_of(cache);
    p.span = {start, counts, start0, q_len};
    p.q = heads_of(q);
    p.o = heads_of(o);
    p.Hq = num_heads;
    p.G = num_heads / cache->num_kv_heads;
    p.rows = (unsigned)rows;
    p.pat = esa::make_pattern(heads, attn_length, layer_idx, num_hidden_layers, head_offset);
    p.scale_log2 = scale * esa::kLog2e;
    p.lse = lse;
    p.err = err;
    // few pairs: the slots of a pair over several warps, up to one chunk of 32 each
    int wpp = 1;
    while (wpp < c4::kAttendWarps && wpp * 32 < attn_length && pairs * wpp < kSms * 16) wpp *= 2;
    p.warps_per_pair = wpp;
    // many pairs: several per warp, as long as every SM has its CTAs
    int ppw = 1;
    while (wpp == 1 && ppw < 4 && pairs >= (int64_t)kSms * 20 * ppw * 4) ppw *= 2;
    p.pairs_per_warp = ppw;
    const dim3 grid((unsigned)ceil_div(rows, c4::kAttendWarps / wpp * ppw), (unsigned)kv);
    return by_head_dim(cache->head_dim, [&](auto d) {
      constexpr int D = decltype(d)::value;
      if (wpp > 1)
        c4::attend_kernel<T, D, true><<<grid, c4::kAttendWarps * 32, 0, (cudaStream_t)stream>>>(p);
      else
        c4::attend_kernel<T, D, false><<<grid, c4::kAttendWarps * 32, 0, (cudaStream_t)stream>>>(p);
      return check_launch(what);
    });
  });
}

}  // extern "C"
