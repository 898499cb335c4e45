/*
 * esa_layer.h -- decoder-layer harness kernels of libesa_b200.so: the
 * memory-bound operations of a pre-norm decoder layer (RMSNorm with a fused
 * residual add, rotary position embedding, SwiGLU, token embedding, per-head
 * query / key norm, activations kept in 8 bits) that surround elastic
 * sparse attention in the C4 decoder-stack configuration.  The reference
 * ships no model code (its module is used inside external decoder layers), so
 * these entry points replace no reference interface; they exist so that the
 * layer around the attention runs without layout copies: RoPE rotates q and k
 * in place inside the QKV projection's output buffer, which the attention
 * kernels then read through strides.
 *
 * Same conventions as esa_b200.h: device pointers owned by the caller, no
 * allocation, launches on `stream`, ESA_OK or a negative code with
 * esa_last_error() describing the failure.  dtype is an esa_dtype_t value
 * (ESA_DTYPE_F32 / _BF16 / _F16); rows are contiguous vectors of `dim`
 * elements (row stride = dim) unless stated otherwise; every pointer is
 * 16-byte aligned and dim * element size is a multiple of 16 bytes.
 * Arithmetic is float32; each output is rounded once to dtype.  Outputs do not
 * overlap inputs or each other unless an entry point allows it.
 */
#ifndef ESA_LAYER_H
#define ESA_LAYER_H

#include <stddef.h>
#include <stdint.h>

#include "esa_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * RMSNorm with an optional residual add:
 *   h = x + residual (residual may be NULL: h = x; h_out may be NULL when
 *       residual is NULL), rounded to dtype and written to h_out;
 *   y = h * rstd * weight,  rstd = 1 / sqrt(mean(h^2) + eps)  (float32,
 *       written to rstd[n_rows]).
 * dim <= 1024 * (16 / element size).
 */
int esa_rmsnorm_forward(int32_t dtype, int64_t n_rows, int32_t dim, const void* x,
                        const void* residual, void* h_out, const void* weight, float eps,
                        void* y, float* rstd, void* stream);

/* Bytes of float32 workspace esa_rmsnorm_backward needs (per-CTA partial
 * sums of the weight gradient). */
size_t esa_rmsnorm_backward_workspace_size(int64_t n_rows, int32_t dim);

/*
 * Backward of esa_rmsnorm_forward given the saved h and rstd:
 *   dh = dh_in + rstd * (weight * dy - xhat * mean(xhat * weight * dy)),
 *        xhat = h * rstd (dh_in, the gradient reaching h from its other
 *        uses, may be NULL);
 *   dweight = sum over rows of dy * xhat (written in dtype).
 * dh may alias dh_in.
 */
int esa_rmsnorm_backward(int32_t dtype, int64_t n_rows, int32_t dim, const void* h,
                         const void* weight, const float* rstd, const void* dy,
                         const void* dh_in, void* dh, void* dweight, void* workspace,
                         size_t workspace_bytes, void* stream);

/*
 * Rotary position embedding, in place, on q [B, Hq, L, D] and k [B, Hk, L, D]
 * (esa_tensor_t strides, D contiguous; k.data may be NULL).  For i < D/2 the
 * pair (x[i], x[i + D/2]) of the row at position p is rotated by
 * angle = f32(p) * inv_freq[i] (one float32 rounding; cos and sin in float32):
 *   x'[i] = x[i] cos - x[i + D/2] sin,  x'[i + D/2] = x[i + D/2] cos + x[i] sin
 * ("rotate half" convention).  inverse != 0 rotates by -angle (the backward:
 * applied to the gradients of the rotated q and k).  positions: device int64
 * [L] shared by the batch, or NULL for 0..L-1.  inv_freq: device float32
 * [D/2], e.g. 1 / base^(2i/D) computed by the caller.
 */
int esa_rope_apply(int32_t dtype, int32_t batch, int64_t seq_len, int32_t head_dim,
                   esa_tensor_t q, int32_t num_q_heads, esa_tensor_t k, int32_t num_k_heads,
                   const int64_t* positions, const float* inv_freq, int32_t inverse,
                   void* stream);

/*
 * SwiGLU on a fused gate/up projection: gate_up rows are [gate (ffn) | up
 * (ffn)] (row stride 2 * ffn); out[r, f] = silu(gate) * up with
 * silu(g) = g / (1 + exp(-g)).  ffn * element size is a multiple of 16 bytes.
 */
int esa_swiglu_forward(int32_t dtype, int64_t n_rows, int32_t ffn, const void* gate_up,
                       void* out, void* stream);

/*
 * Backward of esa_swiglu_forward: dgate_up rows = [dout * up * silu'(gate) |
 * dout * silu(gate)]; out_recomputed (may be NULL) receives the forward
 * output again, for the down projection's weight gradient, in the same pass.
 */
int esa_swiglu_backward(int32_t dtype, int64_t n_rows, int32_t ffn, const void* gate_up,
                        const void* dout, void* dgate_up, void* out_recomputed, void* stream);

/*
 * Token embedding: out[r] = scale * weight[ids[r]] (weight [vocab, dim], out
 * [n_tokens, dim]).  ids: device integers of id_bytes 4 or 8.  An id outside
 * [0, vocab) gives a row of zeros and sets ESA_DEVERR_TOKEN_RANGE.
 * n_tokens <= 2^30, vocab < 2^27.
 */
int esa_embedding_forward(int32_t dtype, int32_t id_bytes, int64_t n_tokens, int64_t vocab,
                          int32_t dim, const void* ids, const void* weight, float scale, void* out,
                          void* stream);

/* Bytes of workspace esa_embedding_backward needs (0 for few tokens). */
size_t esa_embedding_backward_workspace_size(int64_t n_tokens, int64_t vocab, int32_t dim);

/*
 * Gradient of esa_embedding_forward:
 *   dweight[v] = scale * sum over r with ids[r] = v of dy[r]
 * (float32 sums in a fixed order, without atomics: the same in every run;
 * rounded once).  All
 * of dweight [vocab, dim] is written; rows of absent tokens and row
 * padding_idx (none if negative) are zero.  Ids outside [0, vocab) are left
 * out and set ESA_DEVERR_TOKEN_RANGE.  workspace: 256-byte aligned, its
 * contents do not matter; calls in flight at a time need one each.
 */
int esa_embedding_backward(int32_t dtype, int32_t id_bytes, int64_t n_tokens, int64_t vocab,
                           int32_t dim, const void* ids, const void* dy, float scale,
                           int64_t padding_idx, void* dweight, void* workspace,
                           size_t workspace_bytes, void* stream);

/*
 * RMSNorm over each head row of q [B, Hq, L, D] and k [B, Hk, L, D]
 * (esa_tensor_t strides, D contiguous) with a weight of D elements per side,
 * and the rotary embedding of the result, in one pass:
 *   n = x * rstd * weight,  rstd = 1 / sqrt(mean over D of x^2 + eps)
 *   out = n rotated at the row's position ("rotate half", as esa_rope_apply)
 * The angle p * inv_freq[i] is formed in float64 (esa_rope_apply rounds it to
 * float32), so far positions keep their precision.  positions: device int64;
 * entry b * positions_stride_b + l for row l of batch entry b (stride 0:
 * shared by the batch), or NULL for 0..L-1.  num_k_heads 0: no keys (the k
 * arguments are ignored), likewise num_q_heads 0.  q_out / k_out may be q / k
 * themselves (in place), views of a larger buffer such as rows of a key
 * cache, but must not overlap them otherwise.  D: a power of two, 16 to 256
 * (16-bit types) or 8 to 128 (float32).
 */
int esa_qk_norm_rope_forward(int32_t dtype, int32_t batch, int64_t seq_len, int32_t head_dim,
                             esa_tensor_t q, int32_t num_q_heads, esa_tensor_t k,
                             int32_t num_k_heads, const void* q_weight, const void* k_weight,
                             float eps, const int64_t* positions, int64_t positions_stride_b,
                             const float* inv_freq, esa_tensor_t q_out, esa_tensor_t k_out,
                             void* stream);

/* Bytes of workspace esa_qk_norm_rope_backward needs. */
size_t esa_qk_norm_rope_backward_workspace_size(int32_t batch, int64_t seq_len,
                                                int32_t num_q_heads, int32_t num_k_heads,
                                                int32_t head_dim);

/*
 * Backward of esa_qk_norm_rope_forward, given its inputs q, k (before the
 * norm) and the gradients of its outputs:
 *   g = dout rotated back, xhat = x * rstd
 *   dx = rstd * (weight * g - xhat * mean(xhat * weight * g))
 *   dweight = sum over batch, heads and positions of g * xhat   (in dtype)
 * dq / dk may be dq_out / dk_out themselves.  Sums are float32 in a fixed
 * order.  With no rows the weight gradients are zero; so is a given dq_weight
 * / dk_weight of a side without heads.
 */
int esa_qk_norm_rope_backward(int32_t dtype, int32_t batch, int64_t seq_len, int32_t head_dim,
                              esa_tensor_t q, int32_t num_q_heads, esa_tensor_t k,
                              int32_t num_k_heads, const void* q_weight, const void* k_weight,
                              float eps, const int64_t* positions, int64_t positions_stride_b,
                              const float* inv_freq, esa_tensor_t dq_out, esa_tensor_t dk_out,
                              esa_tensor_t dq, esa_tensor_t dk, void* dq_weight, void* dk_weight,
                              void* workspace, size_t workspace_bytes, void* stream);

/*
 * Rows in 8 bits, for activations kept between the forward and the backward
 * pass.  Each group of 128 consecutive elements of a row (the last may be
 * shorter) has a float32 scale s; with a the group's largest magnitude:
 *   ESA_PACK_INT8: s = max(f32(a / 127), 2^-126); code = x / s to the nearest
 *                  integer, ties to even, the quotient taken exactly (int8)
 *   ESA_PACK_E4M3: s = the smallest power of two >= 2^-126 with a <= 448 s;
 *                  code = x / s to the nearest e4m3 value, ties to even (the
 *                  next smaller where code * s passes dtype's largest value)
 * A code stands for code * s.  A group with an infinity or a NaN gets s = NaN
 * and codes 0, so it decodes to NaN.  Every other group decodes to finite values
 * with one exception: where a is the largest float32, 127 * s rounds past it in
 * ESA_PACK_INT8, so codes of 127 decode to infinity there.  codes: n_rows * dim bytes; scales:
 * n_rows * ceil(dim / 128) floats.
 */
#define ESA_PACK_INT8 0
#define ESA_PACK_E4M3 1

int esa_quantize_rows(int32_t dtype, int32_t format, int64_t n_rows, int32_t dim, const void* x,
                      void* codes, float* scales, void* stream);

/* x = code * s in float32, rounded once to dtype (any dtype, not only the one
 * the codes were made from). */
int esa_dequantize_rows(int32_t dtype, int32_t format, int64_t n_rows, int32_t dim,
                        const void* codes, const float* scales, void* x, void* stream);

/* esa_rmsnorm_forward that also writes the 8-bit form of h (as stored in
 * h_out, or of x without a residual) in the same pass.  h_out is the same bit
 * for bit; rstd and y may differ from that entry point's by the order of the
 * float32 sum, so that y is a step of dtype off where that moves its rounding. */
int esa_rmsnorm_pack_forward(int32_t dtype, int32_t format, int64_t n_rows, int32_t dim,
                             const void* x, const void* residual, void* h_out, const void* weight,
                             float eps, void* y, float* rstd, void* codes, float* scales,
                             void* stream);

/* h = the rows that the codes stand for (rounded to dtype), y and rstd the
 * norm of that h: what a backward pass needs of a layer's input, in one pass
 * over the codes. */
int esa_rmsnorm_unpack_forward(int32_t dtype, int32_t format, int64_t n_rows, int32_t dim,
                               const void* codes, const float* scales, const void* weight,
                               float eps, void* h, void* y, float* rstd, void* stream);

/* esa_swiglu_forward (within a rounding: the sigmoid's float32 arithmetic is
 * another) that also writes gate_up in 8 bits.  The gate and the up
 * half of a row are two rows of ffn elements with groups of their own: codes
 * [n_rows, 2, ffn], scales [n_rows, 2, ceil(ffn / 128)]. */
int esa_swiglu_pack_forward(int32_t dtype, int32_t format, int64_t n_rows, int32_t ffn,
                            const void* gate_up, void* out, void* codes, float* scales,
                            void* stream);

/* esa_swiglu_backward from the 8-bit gate_up: gate and up are the float32
 * values code * s; out_recomputed (may be NULL) is the output for them. */
int esa_swiglu_unpack_backward(int32_t dtype, int32_t format, int64_t n_rows, int32_t ffn,
                               const void* codes, const float* scales, const void* dout,
                               void* dgate_up, void* out_recomputed, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* ESA_LAYER_H */
