"""Decoding and scoring with a decoder stack in 4 bits.

The reference attends to keys and values its caller keeps (``cache_position``,
``elastic_sparse_attention.py:728-765``) and ships no model code; this session is
the serving side of :class:`~.decoder.ElasticDecoderStack`: its projections in 4
bits, a :class:`~.cache.PackedKVCache` per layer, a batch of sequences of different
lengths, and answers as log probabilities with alternatives.
"""
from __future__ import annotations

import torch
import torch.nn.functional as F

from . import layer_ops, ops
from .cache import PackedKVCache
from .decoder import ElasticDecoderStack


class PackedDecoder:
    """``batch`` sequences of up to ``max_len`` tokens decoded with the weights of
    ``stack``: projections and LM head kept in 4 bits (``group`` inputs per scale),
    embedding and norms the stack's own.

    :meth:`step` and :meth:`score` take each sequence's next tokens ``input_ids``
    [batch, L] (a prompt, a part of one, or single tokens), ``counts`` [batch] of
    them (default: all; the rest is padding, whose ids are not looked at), and extend
    the caches.  ``lengths``
    (int64 [batch], on the device) holds what has been fed so far.  Nothing is read
    back to the host: a call can be captured into a CUDA graph, whose replays read
    the ids and extend the caches.  Tokens beyond ``max_len`` are left out and set
    ``_lib.DEVERR_KV_RANGE`` and ``_lib.DEVERR_QUERY_RANGE``
    (``ops.device_errors``)."""

    def __init__(self, stack: ElasticDecoderStack, batch: int, max_len: int, group: int = 128):
        if not 1 <= max_len <= stack.max_seq_len:
            raise ValueError(f"max_len {max_len} outside [1, {stack.max_seq_len}]")
        self.stack = stack
        device = stack.embed.device
        with torch.no_grad():
            self.layers = [tuple(layer_ops.quantize_weight4(w, group) for w in
                                 (lw.qkv_proj, lw.o_proj, lw.gate_up_proj, lw.down_proj))
                           for lw in stack.layers]
            self.lm_head = layer_ops.quantize_weight4(stack.lm_head, group)
        self.caches = [PackedKVCache(batch, stack.Hkv, max_len, stack.D, device=device)
                       for _ in stack.layers]
        self.lengths = torch.zeros(batch, dtype=torch.int64, device=device)

    def nbytes(self) -> int:
        """Bytes of the packed weights and the caches."""
        weights = [w for layer in self.layers for w in layer] + [self.lm_head]
        return sum(w.nbytes() for w in weights) + sum(c.nbytes() for c in self.caches)

    def reset(self) -> None:
        """Forget all sequences (the caches' rows are written before they are read)."""
        self.lengths.zero_()

    @staticmethod
    def _project(x: torch.Tensor, weight: layer_ops.PackedWeight4) -> torch.Tensor:
        """x W^T: from the codes for float32 and for few rows of a 16-bit type, else
        with the weight decoded, and rounded to the type, for the call."""
        most = (layer_ops.LINEAR4_MAX_ROWS if x.dtype == torch.float32 else
                layer_ops.LINEAR4_ROWS)
        if x.numel() // x.shape[-1] <= most:
            return layer_ops.linear4(x, weight)
        return torch.matmul(x, layer_ops.dequantize_weight4(weight, x.dtype).t())

    def _check(self, input_ids: torch.Tensor, counts):
        if input_ids.dim() != 2 or input_ids.shape[0] != self.lengths.shape[0]:
            raise ValueError(f"input_ids must be [{self.lengths.shape[0]}, L]")
        if counts is not None:
            if tuple(counts.shape) != tuple(self.lengths.shape):
                raise ValueError("counts must be [batch]")
            counts = counts.to(device=self.lengths.device, dtype=torch.int64)
            counts = counts.clamp(0, input_ids.shape[1])
        return counts

    @torch.no_grad()
    def step(self, input_ids: torch.Tensor, counts: torch.Tensor | None = None) -> torch.Tensor:
        """The final normalised hidden states [batch, L, hidden] of the new tokens
        (rows of padding hold nothing of use)."""
        counts = self._check(input_ids, counts)
        s = self.stack
        B, L = input_ids.shape
        Hq, Hkv, D = s.Hq, s.Hkv, s.D
        if B == 0 or L == 0:
            return s.embed.new_empty(B, L, s.hidden)
        if counts is not None:
            # padding may hold any id: the lookup gets one of the vocabulary
            padding = torch.arange(L, device=counts.device) >= counts[:, None]
            input_ids = input_ids.masked_fill(padding, 0)
        # all tokens of the batch in one row of positions
        positions = (self.lengths[:, None] + torch.arange(L, device=self.lengths.device)).view(-1)
        h = s._embed(input_ids)
        _, y, _ = layer_ops.rmsnorm_forward(h, s._input_norm(0), s.eps)
        for i, (wqkv, wo, wgu, wd) in enumerate(self.layers):
            lw = s.layers[i]
            qkv = self._project(y, wqkv).view(1, B * L, Hq + 2 * Hkv, D)
            q, k = qkv[:, :, :Hq].transpose(1, 2), qkv[:, :, Hq:Hq + Hkv].transpose(1, 2)
            if lw.q_norm is None:
                layer_ops.rope_(q, k, s.inv_freq, positions)
            else:
                layer_ops.qk_norm_rope(q, k, lw.q_norm, lw.k_norm, s.eps, s.inv_freq, positions,
                                       q_out=q, k_out=k)
            x = qkv.view(B, L, Hq + 2 * Hkv, D)
            self.caches[i].write(x[:, :, Hq:Hq + Hkv].transpose(1, 2),
                                 x[:, :, Hq + Hkv:].transpose(1, 2), self.lengths, counts)
            o, _ = ops.forward_packed(x[:, :, :Hq].transpose(1, 2), self.caches[i], s.specs[i],
                                      D ** -0.5, self.lengths, counts)
            a = self._project(o.transpose(1, 2).reshape(B, L, Hq * D), wo)
            h, y, _ = layer_ops.rmsnorm_forward(h, lw.post_attention_norm, s.eps, residual=a)
            m = self._project(layer_ops.swiglu_forward(self._project(y, wgu)), wd)
            h, y, _ = layer_ops.rmsnorm_forward(h, s._input_norm(i + 1), s.eps, residual=m)
        self.lengths += L if counts is None else counts
        return y

    @torch.no_grad()
    def logits(self, hidden: torch.Tensor) -> torch.Tensor:
        """The vocabulary's logits of hidden states [..., hidden] of :meth:`step`."""
        return self._project(hidden.contiguous(), self.lm_head)

    @torch.no_grad()
    def score(self, input_ids: torch.Tensor, counts: torch.Tensor | None = None,
              top_k: int = 0) -> layer_ops.TokenLogProbs:
        """:meth:`step`, and of each new token's row [batch, L] the log probability of
        the token after it in ``input_ids``, the entropy, and the ``top_k`` most
        likely next tokens.  The last token of a sequence has no token after it (log
        probability 0): its alternatives are the next token's."""
        counts = self._check(input_ids, counts)
        layer_ops.check_top_k(top_k, self.lm_head.shape[0])     # before the tokens are fed
        B, L = input_ids.shape
        nxt = F.pad(input_ids[:, 1:], (0, 1), value=layer_ops.IGNORED_TOKEN) if L else input_ids
        if counts is not None:
            after = torch.arange(1, L + 1, device=counts.device) >= counts[:, None]
            nxt = nxt.masked_fill(after, layer_ops.IGNORED_TOKEN)
        y = self.step(input_ids, counts).view(B * L, self.stack.hidden)
        chunk = self.stack.loss_chunk_rows
        parts = [layer_ops.token_logprobs(self.logits(y[r:r + chunk]),
                                          nxt.reshape(-1)[r:r + chunk], top_k=top_k)
                 for r in range(0, max(B * L, 1), chunk)]
        out = []
        for name, tail in (("logprobs", ()), ("entropy", ()), ("stats", (2,)),
                           ("top_ids", (top_k,)), ("top_logprobs", (top_k,))):
            each = [getattr(p, name) for p in parts]
            out.append(None if each[0] is None else
                       (each[0] if len(each) == 1 else torch.cat(each)).view((B, L) + tail))
        return layer_ops.TokenLogProbs(*out)
