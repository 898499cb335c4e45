"""Decoder-layer stack around elastic sparse attention (the C4 configuration).

The reference ships the attention module only (it is meant to sit inside an
external decoder layer), so this harness has no reference counterpart.  It is
a pre-norm Llama-style stack: token embedding, per layer RMSNorm -> fused QKV
projection -> rotary embedding -> elastic sparse attention (layer_idx = layer
number, num_hidden_layers = the stack depth) -> output projection -> residual
add -> RMSNorm -> SwiGLU MLP -> residual add, then a final RMSNorm, the LM
head and the mean next-token cross entropy.

Built for B200 without layout copies:

* The QKV projection writes one [B, L, Hq + 2 Hkv, D] buffer.  RoPE rotates
  its q and k parts in place and the attention kernels read q, k, v straight
  from it through strides; the attention output is written as [B, L, Hq, D],
  the output projection's input, with no transpose.  In the backward the
  attention kernels write dQ, dK, dV into the parts of one gradient buffer of
  the same layout, the inverse rotation runs in place on it, and it feeds the
  projection's weight and input gradients directly (the module path
  ``transpose(1, 2).contiguous()`` of the reference's callers, :244 / :763,
  never happens).
* Residual adds are fused into the following RMSNorm; SwiGLU runs on the
  fused gate/up projection output and recomputes its output in the backward
  instead of keeping it.
* The LM head and loss run over row chunks and produce their gradients in the
  forward, so the [L, vocab] logits never exist in full.
* GEMMs are cuBLAS through torch (bf16 in, fp32 accumulate).

``activation_checkpointing=True`` recomputes each layer in the backward
(keeps only its input), for lengths whose activations do not fit.

Options (all off by default):

* ``embed_scale`` / ``padding_idx``: the token embedding runs in the library's
  lookup (times ``embed_scale``) and its gradient in the sorted-token kernels,
  which leave the row ``padding_idx`` without a gradient; an id outside the
  vocabulary makes its hidden state NaN, and so the loss and the gradients, and
  sets a device error bit, instead of an assert.
* ``qk_norm``: RMSNorm of each query and key head (weights ``q_norm``,
  ``k_norm`` of head_dim) before the rotary embedding, both in one pass; the
  backward normalises again instead of keeping the result.
* ``activation_storage`` = "int8" or "e4m3": what the backward needs is kept
  in 8 bits.  With ``activation_checkpointing`` that is each layer's input
  (written by the norm that precedes the layer, restored together with that
  norm), instead of two full rows; without, the MLP's gate / up rows, the
  largest activation of a layer.  The forward pass works on the activations
  themselves, not on their 8-bit form; its results are within a rounding of
  those without the option (the norm sums in another order, SwiGLU forms its
  sigmoid another way).  Gradients are taken at the decoded values.
"""
from __future__ import annotations

import functools

import torch
import torch.nn as nn
import torch.nn.functional as F
import torch.utils.checkpoint

from . import layer_ops, ops
from .attention import KeyPlanCache, _ensure_monotone
from .layer_ops import PACK_FORMATS, PackedRows
from .ops import PatternSpec


class _NoSecondDerivative(torch.autograd.Function):
    """Gradients as they are, whose own derivative is an error."""

    @staticmethod
    def forward(ctx, root, *grads):
        return tuple(g.detach() for g in grads)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("ElasticDecoderStack has no second derivatives: its gradients are "
                           "computed by kernels that autograd does not see through")


def _first_derivative_only(backward):
    """For a backward made of kernels: under create_graph=True its gradients come
    with a graph that raises when it is used, instead of none or a part of one
    (torch's once_differentiable looks at the incoming gradients alone, and the
    first of those takes none)."""
    @functools.wraps(backward)
    def wrapped(ctx, *grads):
        graph = torch.is_grad_enabled()
        with torch.no_grad():
            out = backward(ctx, *grads)
        if not graph:
            return out
        out = out if isinstance(out, tuple) else (out,)
        root = torch.zeros((), requires_grad=True)
        marked = iter(_NoSecondDerivative.apply(root, *(g for g in out if g is not None)))
        return tuple(None if g is None else next(marked) for g in out)
    return wrapped


class _Embedding(torch.autograd.Function):
    """scale * w[ids]; the row of an id that has none in w starts with a NaN, which
    the norm after it spreads over the row: a step on wrong ids is not silent."""

    @staticmethod
    def forward(ctx, ids, w, scale: float, padding_idx):
        ctx.save_for_backward(ids)
        ctx.meta = (w.shape[0], scale, padding_idx)
        out = layer_ops.embedding_forward(ids, w, scale)
        out[..., 0].masked_fill_((ids < 0) | (ids >= w.shape[0]), float("nan"))
        return out

    @staticmethod
    @_first_derivative_only
    def backward(ctx, dy):
        ids, = ctx.saved_tensors
        vocab, scale, padding_idx = ctx.meta
        return None, layer_ops.embedding_backward(ids, dy, vocab, scale, padding_idx), None, None


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, eps: float):
        x = x.contiguous()
        _, y, rstd = layer_ops.rmsnorm_forward(x, w, eps)
        ctx.save_for_backward(x, w, rstd)
        return y

    @staticmethod
    @_first_derivative_only
    def backward(ctx, dy):
        x, w, rstd = ctx.saved_tensors
        dx, dw = layer_ops.rmsnorm_backward(x, w, rstd, dy)
        return dx, dw, None


class _PackedRMSNorm(torch.autograd.Function):
    """(y, codes, scales) of x: its norm and its 8-bit form, which is what the
    backward keeps of it."""

    @staticmethod
    def forward(ctx, x, w, eps: float, fmt: str):
        ctx.set_materialize_grads(False)     # no zeros for the codes' gradients
        _, y, _, p = layer_ops.rmsnorm_forward_packed(x.contiguous(), w, eps, format=fmt)
        ctx.save_for_backward(p.codes, p.scales, w)
        ctx.meta = (fmt, x.dtype)
        ctx.eps = eps
        ctx.mark_non_differentiable(p.codes, p.scales)
        return y, p.codes, p.scales

    @staticmethod
    @_first_derivative_only
    def backward(ctx, dy, _codes, _scales):
        codes, scales, w = ctx.saved_tensors
        x, _, rstd = layer_ops.rmsnorm_from_packed(PackedRows(codes, scales, *ctx.meta), w, ctx.eps)
        dx, dw = layer_ops.rmsnorm_backward(x, w, rstd, dy)
        return dx, dw, None, None


class _AddRMSNorm(torch.autograd.Function):
    """(h, y) = (a + b, rmsnorm(a + b) * w)."""

    @staticmethod
    def forward(ctx, a, b, w, eps: float):
        h, y, rstd = layer_ops.rmsnorm_forward(a.contiguous(), w, eps, residual=b.contiguous())
        ctx.save_for_backward(h, w, rstd)
        return h, y

    @staticmethod
    @_first_derivative_only
    def backward(ctx, dh, dy):
        h, w, rstd = ctx.saved_tensors
        if dy is None:
            dy = torch.zeros_like(h)
        dx, dw = layer_ops.rmsnorm_backward(h, w, rstd, dy, dh_in=dh)
        return dx, dx, dw, None


class _AttentionBlock(torch.autograd.Function):
    """a = attention(rope(y Wqkv^T)) Wo^T with the layouts described above;
    with q_norm / k_norm, attention(rope(norm(y Wqkv^T)))."""

    @staticmethod
    def forward(ctx, y, wqkv, wo, spec: PatternSpec, heads: tuple, inv_freq, positions,
                plans=None, q_norm=None, k_norm=None, eps: float = 0.0):
        Hq, Hkv, D = heads
        B, L, d = y.shape
        qkv = torch.matmul(y, wqkv.t())                       # [B, L, (Hq + 2 Hkv) D]
        q, k, v = _split_heads(qkv, B, L, Hq, Hkv, D)
        if q_norm is None:
            layer_ops.rope_(q, k, inv_freq, positions)
        else:
            q, k = layer_ops.qk_norm_rope(q, k, q_norm, k_norm, eps, inv_freq, positions)
        scale = D ** -0.5
        probs = ops.probs_buffer(q, k, spec)                  # kept for the backward
        o, lse = ops.forward(q, k, v, spec, scale, probs=probs)   # o: view of [B, L, Hq, D]
        o_rows = o.transpose(1, 2).reshape(B, L, Hq * D)      # a view, no copy
        a = torch.matmul(o_rows, wo.t())
        ctx.save_for_backward(y, wqkv, wo, qkv, o_rows, lse, inv_freq, positions, probs, q_norm,
                              k_norm)
        ctx.meta = (spec, heads, scale, eps)
        ctx.plans = plans
        return a

    @staticmethod
    @_first_derivative_only
    def backward(ctx, da):
        (y, wqkv, wo, qkv, o_rows, lse, inv_freq, positions, probs, q_norm,
         k_norm) = ctx.saved_tensors
        spec, (Hq, Hkv, D), scale, eps = ctx.meta
        B, L, d = y.shape
        da = da.contiguous()
        do_rows = torch.matmul(da, wo)                        # [B, L, Hq D]
        dwo = torch.matmul(da.reshape(-1, d).t(), o_rows.reshape(-1, Hq * D))
        q, k, v = _split_heads(qkv, B, L, Hq, Hkv, D)
        raw_q, raw_k = q, k
        if q_norm is not None:
            q, k = layer_ops.qk_norm_rope(q, k, q_norm, k_norm, eps, inv_freq, positions)
        o = o_rows.view(B, L, Hq, D).transpose(1, 2)
        dqkv = torch.empty_like(qkv)
        dq, dk, dv = _split_heads(dqkv, B, L, Hq, Hkv, D)
        _ensure_monotone(Hq, spec, max(L, 2), y.device)
        plan = ctx.plans.get(q, k, spec) if ctx.plans is not None else None
        ops.backward(q, k, v, o, lse, do_rows.view(B, L, Hq, D).transpose(1, 2), spec, scale,
                     dq=dq, dk=dk, dv=dv, probs=probs, key_plan=plan)
        del do_rows
        dq_norm = dk_norm = None
        if q_norm is None:
            layer_ops.rope_(dq, dk, inv_freq, positions, inverse=True)
        else:
            _, _, dq_norm, dk_norm = layer_ops.qk_norm_rope_backward(
                raw_q, raw_k, q_norm, k_norm, eps, inv_freq, dq, dk, positions, dq=dq, dk=dk)
        dy = torch.matmul(dqkv, wqkv)
        dwqkv = torch.matmul(dqkv.reshape(-1, dqkv.shape[-1]).t(), y.reshape(-1, d))
        return dy, dwqkv, dwo, None, None, None, None, None, dq_norm, dk_norm, None


def _split_heads(qkv, B, L, Hq, Hkv, D):
    """q [B, Hq, L, D], k / v [B, Hkv, L, D] views of a [B, L, (Hq+2Hkv) D] buffer."""
    x = qkv.view(B, L, Hq + 2 * Hkv, D)
    return (x[:, :, :Hq].transpose(1, 2), x[:, :, Hq:Hq + Hkv].transpose(1, 2),
            x[:, :, Hq + Hkv:].transpose(1, 2))


class _MLPBlock(torch.autograd.Function):
    """out = swiglu(y Wgu^T) Wd^T, rows of Wgu = [gate; up]."""

    @staticmethod
    def forward(ctx, y, wgu, wd):
        gu = torch.matmul(y, wgu.t())
        m = layer_ops.swiglu_forward(gu)
        out = torch.matmul(m, wd.t())
        ctx.save_for_backward(y, wgu, wd, gu)
        return out

    @staticmethod
    @_first_derivative_only
    def backward(ctx, dout):
        y, wgu, wd, gu = ctx.saved_tensors
        d = y.shape[-1]
        dout = dout.contiguous()
        dm = torch.matmul(dout, wd)
        dgu, m = layer_ops.swiglu_backward(gu, dm, recompute=True)
        del dm
        dwd = torch.matmul(dout.reshape(-1, d).t(), m.reshape(-1, m.shape[-1]))
        del m
        dy = torch.matmul(dgu, wgu)
        dwgu = torch.matmul(dgu.reshape(-1, dgu.shape[-1]).t(), y.reshape(-1, d))
        return dy, dwgu, dwd


class _PackedMLPBlock(torch.autograd.Function):
    """:class:`_MLPBlock` whose gate / up rows are kept in 8 bits."""

    @staticmethod
    def forward(ctx, y, wgu, wd, fmt: str):
        m, p = layer_ops.swiglu_forward_packed(torch.matmul(y, wgu.t()), fmt)
        ctx.save_for_backward(y, wgu, wd, p.codes, p.scales)
        ctx.meta = (fmt, m.dtype)
        return torch.matmul(m, wd.t())

    @staticmethod
    @_first_derivative_only
    def backward(ctx, dout):
        y, wgu, wd, codes, scales = ctx.saved_tensors
        d = y.shape[-1]
        dout = dout.contiguous()
        dm = torch.matmul(dout, wd)
        dgu, m = layer_ops.swiglu_backward_packed(PackedRows(codes, scales, *ctx.meta), dm)
        del dm
        dwd = torch.matmul(dout.reshape(-1, d).t(), m.reshape(-1, m.shape[-1]))
        del m
        dy = torch.matmul(dgu, wgu)
        dwgu = torch.matmul(dgu.reshape(-1, dgu.shape[-1]).t(), y.reshape(-1, d))
        return dy, dwgu, dwd, None


class _PackedLayer(torch.autograd.Function):
    """A decoder layer of which nothing but its input in 8 bits is kept, up to its
    last residual add: (h', m) with h' + m what :class:`_PackedLayerNorm` takes.
    That class's backward runs the layer again and leaves the run in ``run`` (a
    list that the two share) for the backward here to differentiate: as two
    nodes, because a node's incoming gradients live until it returns, and the
    norm's two rows per token are not needed while the layer runs backward."""

    @staticmethod
    def forward(ctx, run: list, stack, i: int, h, y, positions, *weights):
        ctx.run = run
        h, m = stack._layer_body(i, h, y, positions, weights)
        return h.contiguous(), m.contiguous()

    @staticmethod
    @_first_derivative_only
    def backward(ctx, dh, dm):
        edges, wanted, wants = ctx.run.pop()
        grads = iter(torch.autograd.grad(edges, wanted, (dh, dm)))
        gh, gy = next(grads), next(grads)
        return (None, None, None, gh, gy, None,
                *(next(grads) if want else None for want in wants))


class _PackedLayerNorm(torch.autograd.Function):
    """The add and norm after a :class:`_PackedLayer`: (h', y', codes', scales'),
    codes' / scales' the 8-bit form of h' = h + m (None after the last layer).
    The backward restores the layer's input h and y = norm(h) from its codes and
    runs the layer again, with the format and the weights of the forward pass.
    ``layer``: (codes, scales, positions, weight of the norm before the layer,
    the layer's own weights)."""

    @staticmethod
    def forward(ctx, run: list, stack, i: int, fmt: str, h, m, next_norm, layer: tuple):
        ctx.set_materialize_grads(False)     # no zeros for the codes' gradients
        ctx.run, ctx.stack, ctx.i, ctx.meta = run, stack, i, (fmt, h.dtype)
        ctx.save_for_backward(next_norm, *layer)
        if i + 1 == len(stack.layers):       # no layer follows that would keep h
            h, y, _ = layer_ops.rmsnorm_forward(h, next_norm, stack.eps, residual=m)
            return h, y, None, None
        h, y, _, p = layer_ops.rmsnorm_forward_packed(h, next_norm, stack.eps, residual=m,
                                                      format=fmt)
        ctx.mark_non_differentiable(p.codes, p.scales)
        return h, y, p.codes, p.scales

    @staticmethod
    @_first_derivative_only
    def backward(ctx, dh, dy, _codes, _scales):
        next_norm, codes, scales, positions, input_norm, *weights = ctx.saved_tensors
        stack = ctx.stack
        h, y, _ = layer_ops.rmsnorm_from_packed(PackedRows(codes, scales, *ctx.meta), input_norm,
                                                stack.eps)
        below = ctx.needs_input_grad[4]      # the layer runs backward too
        wants = [w is not None and w.requires_grad for w in weights]
        wanted = [h.requires_grad_(), y.requires_grad_()]
        wanted += [w for w, want in zip(weights, wants) if want]
        with torch.set_grad_enabled(below):
            h, m = stack._layer_body(ctx.i, h, y, positions, weights)
        if below:
            edges = [torch.autograd.graph.get_gradient_edge(t) for t in (h, m)]
            ctx.run[:] = [(edges, wanted, wants)]
            # a call that asks for gradients above this layer alone never takes it
            torch.autograd.Variable._execution_engine.queue_callback(ctx.run.clear)
        del wanted
        h, _, rstd = layer_ops.rmsnorm_forward(h.detach(), next_norm, stack.eps,
                                               residual=m.detach())
        del y, m
        if dy is None:
            dy = torch.zeros_like(h)
        ds, dw = layer_ops.rmsnorm_backward(h, next_norm, rstd, dy, dh_in=dh)
        return None, None, None, None, ds, ds, dw if next_norm.requires_grad else None, None


class _LMHeadCrossEntropy(torch.autograd.Function):
    """Mean cross entropy of softmax(y W^T) against targets (-100 = ignored),
    over row chunks; the gradients are formed in the forward."""

    @staticmethod
    def forward(ctx, y, w, targets, chunk: int):
        d = y.shape[-1]
        y2 = y.reshape(-1, d)
        t = targets.reshape(-1)
        n = y2.shape[0]
        dy = torch.empty_like(y2)
        dw = torch.zeros(w.shape, dtype=torch.float32, device=w.device)
        loss_sum = torch.zeros((), dtype=torch.float32, device=y.device)
        count = (t != -100).sum()
        for s in range(0, n, chunk):
            yc, tc = y2[s:s + chunk], t[s:s + chunk]
            logits = torch.matmul(yc, w.t()).float()
            lse = torch.logsumexp(logits, dim=-1)
            valid = tc != -100
            tcl = tc.clamp_min(0)
            tgt = logits.gather(1, tcl[:, None])[:, 0]
            loss_sum += ((lse - tgt) * valid).sum()
            p = logits.sub_(lse[:, None]).exp_()              # softmax, in place
            p[torch.arange(p.shape[0], device=p.device), tcl] -= 1.0
            p.mul_(valid[:, None])
            g = p.to(y.dtype)
            del p, logits
            dy[s:s + chunk] = torch.matmul(g, w)
            dw += torch.matmul(g.t(), yc).float()
        inv = 1.0 / count.clamp_min(1).float()
        ctx.save_for_backward(dy, dw, inv)
        ctx.shape = y.shape
        ctx.w_dtype = w.dtype
        return loss_sum * inv

    @staticmethod
    @_first_derivative_only
    def backward(ctx, dloss):
        dy, dw, inv = ctx.saved_tensors
        s = dloss * inv
        return (dy * s.to(dy.dtype)).view(ctx.shape), (dw * s).to(ctx.w_dtype), None, None


class _LMHeadLogProbs(torch.autograd.Function):
    """(log probabilities of ``tokens`` (-100: 0), entropies) of softmax(y W^T), over
    row chunks; the backward forms each chunk's logits again."""

    @staticmethod
    def forward(ctx, y, w, tokens, chunk: int):
        ctx.set_materialize_grads(False)
        y2, t = y.reshape(-1, y.shape[-1]), tokens.reshape(-1)
        parts = [layer_ops.token_logprobs(torch.matmul(y2[s:s + chunk], w.t()), t[s:s + chunk])
                 for s in range(0, y2.shape[0], chunk)]
        logprobs, entropy, stats = (
            torch.cat([getattr(p, name) for p in parts]) if parts
            else torch.empty((0,) + tail, device=y.device)
            for name, tail in (("logprobs", ()), ("entropy", ()), ("stats", (2,))))
        ctx.save_for_backward(y, w, tokens, entropy, stats)
        ctx.chunk = chunk
        # entropy is saved: what is returned is another tensor, so that writing to it
        # does not reach the backward
        return logprobs.view(tokens.shape), entropy.clone().view(tokens.shape)

    @staticmethod
    @_first_derivative_only
    def backward(ctx, dlogprobs, dentropy):
        y, w, tokens, entropy, stats = ctx.saved_tensors
        y2, t, chunk = y.reshape(-1, y.shape[-1]), tokens.reshape(-1), ctx.chunk
        rows = [None if g is None else g.reshape(-1).float() for g in (dlogprobs, dentropy)]
        dy = torch.empty_like(y2)
        dw = torch.zeros(w.shape, dtype=torch.float32, device=w.device)
        for s in range(0, y2.shape[0], chunk):
            part = slice(s, s + chunk)
            logits = torch.matmul(y2[part], w.t())
            scores = layer_ops.TokenLogProbs(None, entropy[part], stats[part], None, None)
            g = layer_ops.token_logprobs_backward(
                logits, t[part], scores, *(None if r is None else r[part] for r in rows), out=logits)
            dy[part] = torch.matmul(g, w)
            dw += torch.matmul(g.t(), y2[part]).float()
        return dy.view(y.shape), dw.to(w.dtype), None, None


class ElasticDecoderLayerWeights(nn.Module):
    """The parameters of one decoder layer (pre-norm, fused QKV and gate/up)."""

    def __init__(self, hidden: int, Hq: int, Hkv: int, D: int, ffn: int, dtype, device,
                 qk_norm: bool = False):
        super().__init__()
        kw = dict(dtype=dtype, device=device)
        self.input_norm = nn.Parameter(torch.ones(hidden, **kw))
        self.qkv_proj = nn.Parameter(torch.empty((Hq + 2 * Hkv) * D, hidden, **kw))
        self.o_proj = nn.Parameter(torch.empty(hidden, Hq * D, **kw))
        self.post_attention_norm = nn.Parameter(torch.ones(hidden, **kw))
        self.gate_up_proj = nn.Parameter(torch.empty(2 * ffn, hidden, **kw))
        self.down_proj = nn.Parameter(torch.empty(hidden, ffn, **kw))
        self.q_norm = nn.Parameter(torch.ones(D, **kw)) if qk_norm else None
        self.k_norm = nn.Parameter(torch.ones(D, **kw)) if qk_norm else None


class ElasticDecoderStack(nn.Module):
    """Token ids -> next-token loss (or final hidden states) through
    ``num_hidden_layers`` decoder layers with elastic sparse attention.

    Defaults are the C4 configuration: 4 layers, hidden 4096, 32 heads of
    128, SwiGLU 11008, RoPE base 10000, vocabulary 32000, attention_length 64.
    Weights are random N(0, 0.02) (norm weights 1) in ``dtype``.  The options
    ``embed_scale``, ``padding_idx``, ``qk_norm`` and ``activation_storage`` are
    described at the top of this file.
    """

    def __init__(self, vocab_size: int = 32000, hidden_size: int = 4096,
                 num_hidden_layers: int = 4, num_attention_heads: int = 32,
                 num_key_value_heads: int | None = None, head_dim: int | None = None,
                 intermediate_size: int = 11008, rope_theta: float = 10000.0,
                 rms_norm_eps: float = 1e-6, attention_length: int = 64,
                 max_seq_len: int = 262144, activation_checkpointing: bool = False,
                 loss_chunk_rows: int = 8192, dtype=torch.bfloat16, device=None, seed: int = 0,
                 embed_scale: float | None = None, padding_idx: int | None = None,
                 qk_norm: bool = False, activation_storage: str | None = None):
        super().__init__()
        if activation_storage is not None and activation_storage not in PACK_FORMATS:
            raise ValueError(f"activation_storage must be one of {sorted(PACK_FORMATS)} or None")
        if padding_idx is not None and not 0 <= padding_idx < vocab_size:
            raise ValueError(f"padding_idx {padding_idx} outside [0, {vocab_size})")
        self.embed_scale = embed_scale
        self.padding_idx = padding_idx
        self.activation_storage = activation_storage
        self.Hq = num_attention_heads
        self.Hkv = num_key_value_heads or num_attention_heads
        if self.Hq % self.Hkv:
            raise ValueError("num_attention_heads must be divisible by num_key_value_heads")
        self.D = head_dim or hidden_size // num_attention_heads
        self.hidden = hidden_size
        self.ffn = intermediate_size
        self.eps = rms_norm_eps
        self.max_seq_len = max_seq_len
        self.checkpointing = activation_checkpointing
        self.loss_chunk_rows = loss_chunk_rows
        self.specs = [PatternSpec(i, num_hidden_layers, attention_length)
                      for i in range(num_hidden_layers)]
        # per layer: the backward's key plan for the current shapes
        self.key_plans = [KeyPlanCache() for _ in range(num_hidden_layers)]
        kw = dict(dtype=dtype, device=device)
        self.embed = nn.Parameter(torch.empty(vocab_size, hidden_size, **kw))
        self.layers = nn.ModuleList(
            ElasticDecoderLayerWeights(hidden_size, self.Hq, self.Hkv, self.D, intermediate_size,
                                       dtype, device, qk_norm) for _ in range(num_hidden_layers))
        self.final_norm = nn.Parameter(torch.ones(hidden_size, **kw))
        self.lm_head = nn.Parameter(torch.empty(vocab_size, hidden_size, **kw))
        self.register_buffer("inv_freq", layer_ops.rope_inv_freq(self.D, rope_theta, device),
                             persistent=False)
        g = torch.Generator(device="cpu").manual_seed(seed)
        with torch.no_grad():
            for p in self.parameters():
                if p.dim() == 2:
                    p.copy_(torch.randn(p.shape, generator=g) * 0.02)

    def _input_norm(self, i: int) -> nn.Parameter:
        """The weight of the norm before layer i (the final norm after the last)."""
        return self.layers[i].input_norm if i < len(self.layers) else self.final_norm

    def _layer_weights(self, i: int) -> list:
        """What layer i multiplies with, in the order :meth:`_layer_body` takes it (the
        query / key norms None without ``qk_norm``); then the weights of the norms
        before and after the layer."""
        lw = self.layers[i]
        return [lw.qkv_proj, lw.o_proj, lw.q_norm, lw.k_norm, lw.post_attention_norm,
                lw.gate_up_proj, lw.down_proj, self._input_norm(i), self._input_norm(i + 1)]

    def _layer_body(self, i: int, h, y, positions, weights, mlp_format: str | None = None):
        """Layer i up to its last residual add: (h, m), whose sum the next norm
        takes.  ``mlp_format``: keep the gate / up rows in that 8-bit format."""
        qkv_proj, o_proj, q_norm, k_norm, post_attention_norm, gate_up_proj, down_proj = weights
        a = _AttentionBlock.apply(y, qkv_proj, o_proj, self.specs[i],
                                  (self.Hq, self.Hkv, self.D), self.inv_freq, positions,
                                  self.key_plans[i], q_norm, k_norm, self.eps)
        h, y2 = _AddRMSNorm.apply(h, a, post_attention_norm, self.eps)
        if mlp_format is not None:
            m = _PackedMLPBlock.apply(y2, gate_up_proj, down_proj, mlp_format)
        else:
            m = _MLPBlock.apply(y2, gate_up_proj, down_proj)
        return h, m

    def _layer(self, i: int, h, y, positions):
        *of_layer, _, next_norm = self._layer_weights(i)
        keeps = not self.checkpointing and torch.is_grad_enabled()
        h, m = self._layer_body(i, h, y, positions, of_layer,
                                self.activation_storage if keeps else None)
        return _AddRMSNorm.apply(h, m, next_norm, self.eps)

    def _embed(self, ids):
        if self.embed_scale is None and self.padding_idx is None:
            return F.embedding(ids, self.embed)
        return _Embedding.apply(ids, self.embed,
                                1.0 if self.embed_scale is None else self.embed_scale,
                                self.padding_idx)

    def forward(self, input_ids: torch.Tensor, labels: torch.Tensor | None = None,
                positions: torch.Tensor | None = None):
        """input_ids [B, L] -> mean next-token cross entropy against labels
        (shifted by one, -100 ignored), or the final normalised hidden states
        [B, L, hidden] when labels is None."""
        B, L = input_ids.shape
        if L > self.max_seq_len:
            raise ValueError(f"sequence length {L} exceeds max_seq_len {self.max_seq_len}")
        if positions is None:
            positions = torch.arange(L, device=input_ids.device)
        h = self._embed(input_ids)
        if self.checkpointing and self.activation_storage is not None and torch.is_grad_enabled():
            y, codes, scales = _PackedRMSNorm.apply(h, self._input_norm(0), self.eps,
                                                    self.activation_storage)
            for i in range(len(self.layers)):
                *weights, input_norm, next_norm = self._layer_weights(i)
                run = []
                layer = (codes, scales, positions, input_norm, *weights)
                h, m = _PackedLayer.apply(run, self, i, h, y, positions, *weights)
                h, y, codes, scales = _PackedLayerNorm.apply(
                    run, self, i, self.activation_storage, h, m, next_norm, layer)
                del m
        else:
            y = _RMSNorm.apply(h, self._input_norm(0), self.eps)
            for i in range(len(self.layers)):
                if self.checkpointing and torch.is_grad_enabled():
                    h, y = torch.utils.checkpoint.checkpoint(self._layer, i, h, y, positions,
                                                             use_reentrant=False)
                else:
                    h, y = self._layer(i, h, y, positions)
        if labels is None:
            return y
        targets = torch.full_like(labels, -100)
        targets[:, :-1] = labels[:, 1:]
        return _LMHeadCrossEntropy.apply(y, self.lm_head, targets, self.loss_chunk_rows)

    def token_logprobs(self, input_ids: torch.Tensor, labels: torch.Tensor | None = None,
                       positions: torch.Tensor | None = None):
        """(log probabilities, entropies), float32 [B, L]: of each row's next token in
        ``labels`` (shifted by one as in :meth:`forward`, -100 ignored: 0; default:
        ``input_ids``), and of the row's distribution over the vocabulary.  The last
        row of a sequence has no next token: 0 and its entropy.  Both are
        differentiable (policy gradients, distillation); the [L, vocab] logits exist
        ``loss_chunk_rows`` rows at a time, in the backward again."""
        labels = input_ids if labels is None else labels
        if labels.shape != input_ids.shape:
            raise ValueError(f"labels {list(labels.shape)} must be shaped like input_ids "
                             f"{list(input_ids.shape)}")
        targets = torch.full_like(labels, layer_ops.IGNORED_TOKEN)
        targets[:, :-1] = labels[:, 1:]
        return _LMHeadLogProbs.apply(self(input_ids, positions=positions), self.lm_head, targets,
                                     self.loss_chunk_rows)

    def flops_per_token(self, seq_len: int) -> float:
        """Dense GEMM FLOPs per token of one forward + backward (3 x 2 x
        params in the projections and the LM head), without attention."""
        d, f = self.hidden, self.ffn
        per_layer = d * (self.Hq + 2 * self.Hkv) * self.D + self.Hq * self.D * d + 3 * d * f
        return 6.0 * (len(self.layers) * per_layer + self.lm_head.shape[0] * d)
