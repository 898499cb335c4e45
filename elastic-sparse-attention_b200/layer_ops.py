"""Tensor-level calls of the decoder-layer harness kernels (include/esa_layer.h):
RMSNorm with a fused residual add, rotary embedding in place, SwiGLU, token
embedding and its gradient, per-head query / key norm with the rotary
embedding, rows kept in 8 bits between forward and backward, log probabilities
of tokens and their gradient, products with weights in 4 bits.

Like ``ops``, torch only allocates memory and provides the stream; every
kernel is in libesa_b200.so and there is no fallback.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _lib
from .ops import _check_device, _on


def _dtype_code(t: torch.Tensor) -> int:
    if t.dtype not in _lib.DTYPES:
        raise TypeError(f"unsupported dtype {t.dtype}")
    return _lib.DTYPES[t.dtype]


def _shape(t: torch.Tensor) -> tuple:
    """The shape of a row operand; its last axis is the feature axis."""
    if t.dim() == 0:
        raise ValueError("row operands need a feature axis")
    return tuple(t.shape)


def _rows(t: torch.Tensor, dim: int) -> int:
    if not t.is_contiguous() or t.shape[-1] != dim:
        raise ValueError("row operands must be contiguous with the feature axis last")
    if dim == 0:
        raise ValueError("rows need at least one element")
    return t.numel() // dim


def rmsnorm_forward(x: torch.Tensor, weight: torch.Tensor, eps: float,
                    residual: torch.Tensor | None = None):
    """(h, y, rstd): h = x + residual (x itself without a residual), y =
    h * rstd * weight, rstd float32 per row."""
    dev = _check_device(x, weight)
    dim = x.shape[-1]
    n = _rows(x, dim)
    y = torch.empty_like(x)
    rstd = torch.empty(x.shape[:-1], dtype=torch.float32, device=dev)
    h = x
    if residual is not None:
        if residual.shape != x.shape or residual.dtype != x.dtype:
            raise ValueError("residual must match x")
        _rows(residual, dim)
        h = torch.empty_like(x)
    lib = _lib.load()
    with _on(dev):
        _lib.check(lib.esa_rmsnorm_forward(
            _dtype_code(x), n, dim, x.data_ptr(), _lib.ptr(residual),
            h.data_ptr() if residual is not None else None, weight.data_ptr(), eps,
            y.data_ptr(), rstd.data_ptr(), _lib.stream_handle(dev)), "esa_rmsnorm_forward")
    return h, y, rstd


def rmsnorm_backward(h: torch.Tensor, weight: torch.Tensor, rstd: torch.Tensor,
                     dy: torch.Tensor, dh_in: torch.Tensor | None = None):
    """(dh, dweight) of :func:`rmsnorm_forward`; dh includes dh_in."""
    dev = _check_device(h, weight, rstd, dy)
    dim = h.shape[-1]
    n = _rows(h, dim)
    dy = dy.contiguous()
    if dh_in is not None:
        dh_in = dh_in.contiguous()
    dh = torch.empty_like(h)
    dw = torch.empty_like(weight)
    lib = _lib.load()
    need = lib.esa_rmsnorm_backward_workspace_size(n, dim)
    ws = torch.empty(max(int(need), 16), dtype=torch.uint8, device=dev)
    with _on(dev):
        _lib.check(lib.esa_rmsnorm_backward(
            _dtype_code(h), n, dim, h.data_ptr(), weight.data_ptr(), rstd.data_ptr(),
            dy.data_ptr(), _lib.ptr(dh_in), dh.data_ptr(), dw.data_ptr(), ws.data_ptr(),
            ws.numel(), _lib.stream_handle(dev)), "esa_rmsnorm_backward")
    return dh, dw


def rope_inv_freq(head_dim: int, base: float, device) -> torch.Tensor:
    """1 / base^(2i / head_dim) for i < head_dim / 2, float32 (the usual
    Llama-style table: integer exponents 0, 2, ... divided by head_dim)."""
    exps = torch.arange(0, head_dim, 2, dtype=torch.int64).float() / head_dim
    return (1.0 / (base ** exps)).to(device=device, dtype=torch.float32)


def _check_inv_freq(inv_freq: torch.Tensor, head_dim: int) -> None:
    if (inv_freq.dtype != torch.float32 or inv_freq.numel() != head_dim // 2
            or not inv_freq.is_contiguous()):
        raise ValueError("inv_freq must be float32 [head_dim / 2]")


def rope_(q: torch.Tensor, k: torch.Tensor | None, inv_freq: torch.Tensor,
          positions: torch.Tensor | None = None, inverse: bool = False) -> None:
    """Rotate q [B, Hq, L, D] and k [B, Hk, L, D] (strided views with a
    contiguous D axis, e.g. parts of a QKV projection buffer) in place.
    ``inverse`` rotates back (the backward, applied to gradients)."""
    dev = _check_device(q, inv_freq)
    B, Hq, L, D = q.shape
    if k is not None and (k.shape[0] != B or k.shape[2] != L or k.shape[3] != D or
                          k.dtype != q.dtype):
        raise ValueError("q and k must share batch, length, head_dim and dtype")
    _check_inv_freq(inv_freq, D)
    if positions is not None:
        positions = positions.to(device=dev, dtype=torch.int64).contiguous()
        if positions.numel() != L:
            raise ValueError("positions must hold one entry per row")
    empty = _lib.EsaTensor(None, 0, 0, 0)
    lib = _lib.load()
    with _on(dev):
        _lib.check(lib.esa_rope_apply(
            _dtype_code(q), B, L, D, _lib.tensor4(q), Hq,
            _lib.tensor4(k) if k is not None else empty, k.shape[1] if k is not None else 0,
            _lib.ptr(positions), inv_freq.data_ptr(), 1 if inverse else 0,
            _lib.stream_handle(dev)), "esa_rope_apply")


def swiglu_forward(gate_up: torch.Tensor) -> torch.Tensor:
    """silu(gate) * up for rows [gate | up] of width 2 * ffn."""
    dev = _check_device(gate_up)
    ffn = gate_up.shape[-1] // 2
    n = _rows(gate_up, 2 * ffn)
    out = torch.empty(gate_up.shape[:-1] + (ffn,), dtype=gate_up.dtype, device=dev)
    lib = _lib.load()
    with _on(dev):
        _lib.check(lib.esa_swiglu_forward(_dtype_code(gate_up), n, ffn, gate_up.data_ptr(),
                                          out.data_ptr(), _lib.stream_handle(dev)),
                   "esa_swiglu_forward")
    return out


def swiglu_backward(gate_up: torch.Tensor, dout: torch.Tensor, recompute: bool = True):
    """(d gate_up, forward output recomputed or None)."""
    dev = _check_device(gate_up, dout)
    ffn = gate_up.shape[-1] // 2
    n = _rows(gate_up, 2 * ffn)
    dout = dout.contiguous()
    dgu = torch.empty_like(gate_up)
    out = (torch.empty(gate_up.shape[:-1] + (ffn,), dtype=gate_up.dtype, device=dev)
           if recompute else None)
    lib = _lib.load()
    with _on(dev):
        _lib.check(lib.esa_swiglu_backward(_dtype_code(gate_up), n, ffn, gate_up.data_ptr(),
                                           dout.data_ptr(), dgu.data_ptr(), _lib.ptr(out),
                                           _lib.stream_handle(dev)), "esa_swiglu_backward")
    return dgu, out


# ---------------------------------------------------------------------------
# Token embedding
# ---------------------------------------------------------------------------
def _empty(shape, dtype: torch.dtype, dev: torch.device) -> torch.Tensor:
    """torch.empty of a contiguous tensor; with the strides given torch takes a
    third less host time, which single-token calls feel."""
    strides, n = [], 1
    for d in reversed(shape):
        strides.append(n)
        n *= d if d > 1 else 1
    strides.reverse()
    return torch.empty_strided(shape, strides, dtype=dtype, device=dev)


def _ids(ids: torch.Tensor) -> torch.Tensor:
    if ids.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"token ids must be int64 or int32, got {ids.dtype}")
    return ids.contiguous()


def embedding_forward(ids: torch.Tensor, weight: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """scale * weight[ids], [*ids.shape, dim], rounded once.  An id outside
    [0, vocab) gives a row of zeros and sets ``_lib.DEVERR_TOKEN_RANGE`` in
    the device error word (``ops.device_errors``); no host round trip."""
    dev = _check_device(ids, weight)
    ids = _ids(ids)
    if weight.dim() != 2:
        raise ValueError("weight must be [vocab, dim]")
    vocab, dim = weight.shape
    _rows(weight, dim)
    out = _empty(tuple(ids.shape) + (dim,), weight.dtype, dev)
    _lib.launch(_lib.load().esa_embedding_forward, dev, _dtype_code(weight), ids.element_size(),
                ids.numel(), vocab, dim, ids.data_ptr(), weight.data_ptr(), scale, out.data_ptr())
    return out


def embedding_backward(ids: torch.Tensor, dy: torch.Tensor, vocab_size: int, scale: float = 1.0,
                       padding_idx: int | None = None) -> torch.Tensor:
    """dweight [vocab_size, dim] of :func:`embedding_forward` for dy
    [*ids.shape, dim]: float32 sums over each token's rows in a fixed order
    (the same in every run), rounded once to dy's dtype.  Rows of absent
    tokens and the row ``padding_idx`` are zero."""
    dev = _check_device(ids, dy)
    ids = _ids(ids)
    dim = dy.shape[-1]
    if dy.shape[:-1] != ids.shape:
        raise ValueError("dy must be [*ids.shape, dim]")
    if padding_idx is not None and not 0 <= padding_idx < vocab_size:
        raise ValueError(f"padding_idx {padding_idx} outside [0, {vocab_size})")
    code = _dtype_code(dy)
    dy = dy.contiguous()
    dw = _empty((vocab_size, dim), dy.dtype, dev)
    lib = _lib.load()
    n = ids.numel()
    need = lib.esa_embedding_backward_workspace_size(n, vocab_size, dim)
    ws = _empty((need,), torch.uint8, dev) if need else None
    _lib.launch(lib.esa_embedding_backward, dev, code, ids.element_size(), n, vocab_size, dim,
                ids.data_ptr(), dy.data_ptr(), scale, -1 if padding_idx is None else padding_idx,
                dw.data_ptr(), _lib.ptr(ws), need)
    return dw


# ---------------------------------------------------------------------------
# Query / key norm with the rotary embedding
# ---------------------------------------------------------------------------
_NO_TENSOR = _lib.EsaTensor(None, 0, 0, 0)


def _t4(t: torch.Tensor | None) -> _lib.EsaTensor:
    return _NO_TENSOR if t is None else _lib.tensor4(t)


def _check_head_weight(name: str, w, like: torch.Tensor, dev: torch.device) -> None:
    if (w is None or w.shape != like.shape[-1:] or w.dtype != like.dtype or w.device != dev
            or not w.is_contiguous()):
        raise ValueError(f"{name}_weight must be a contiguous [head_dim] tensor of q's dtype and "
                         "device")


def _qk_checks(q, k, q_weight, k_weight, inv_freq, positions):
    """(device, B, Hq, Hk, L, D, positions, their batch stride)."""
    dev = _check_device(q, inv_freq)
    B, Hq, L, D = q.shape
    _check_head_weight("q", q_weight, q, dev)
    Hk = 0
    if k is not None:
        kB, Hk, kL, kD = k.shape
        if kB != B or kL != L or kD != D or k.dtype != q.dtype or k.device != dev:
            raise ValueError("q and k must share batch, length, head_dim, dtype and device")
        _check_head_weight("k", k_weight, k, dev)
    _check_inv_freq(inv_freq, D)
    stride = 0
    if positions is not None:
        shape = tuple(positions.shape)
        if shape != (L,) and shape != (B, L):
            raise ValueError("positions must be [L] or [B, L]")
        if positions.dtype != torch.int64 or positions.device != dev:
            positions = positions.to(device=dev, dtype=torch.int64)
        positions = positions.contiguous()
        stride = L if len(shape) == 2 else 0
    return dev, B, Hq, Hk, L, D, positions, stride


def _heads_out(name: str, out: torch.Tensor | None, x: torch.Tensor) -> torch.Tensor:
    """``out`` if it fits x [B, H, L, D]; by default a new tensor whose heads
    of a token lie side by side (storage [B, L, H, D])."""
    if out is None:
        B, H, L, D = x.shape
        return torch.empty_strided((B, H, L, D), (L * H * D, D, H * D, 1), dtype=x.dtype,
                                   device=x.device)
    if out.shape != x.shape or out.dtype != x.dtype or out.device != x.device:
        raise ValueError(f"{name} must match its input's shape, dtype and device")
    return out


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor | None, q_weight: torch.Tensor,
                 k_weight: torch.Tensor | None, eps: float, inv_freq: torch.Tensor,
                 positions: torch.Tensor | None = None, q_out: torch.Tensor | None = None,
                 k_out: torch.Tensor | None = None):
    """(q', k'): each head row of q [B, Hq, L, D] and k [B, Hk, L, D] (strided
    views with a contiguous D axis; k may be None) RMS-normalised with its
    side's [D] weight, then rotated at its position, in one pass.  positions:
    [L] shared by the batch, [B, L], or None for 0 .. L-1.  ``q_out`` /
    ``k_out`` receive the result (e.g. rows of a key cache; q / k themselves
    for in place); by default new [B, H, L, D] views of [B, L, H, D] storage."""
    dev, B, Hq, Hk, L, D, positions, stride = _qk_checks(q, k, q_weight, k_weight, inv_freq,
                                                         positions)
    q_out = _heads_out("q_out", q_out, q)
    if k is not None:
        k_out = _heads_out("k_out", k_out, k)
    elif k_out is not None:
        raise ValueError("k_out without k")
    _lib.launch(_lib.load().esa_qk_norm_rope_forward, dev, _dtype_code(q), B, L, D, _t4(q), Hq,
                _t4(k), Hk, q_weight.data_ptr(), _lib.ptr(k_weight), eps, _lib.ptr(positions),
                stride, inv_freq.data_ptr(), _t4(q_out), _t4(k_out))
    return q_out, k_out


def qk_norm_rope_backward(q: torch.Tensor, k: torch.Tensor | None, q_weight: torch.Tensor,
                          k_weight: torch.Tensor | None, eps: float, inv_freq: torch.Tensor,
                          dq_out: torch.Tensor, dk_out: torch.Tensor | None,
                          positions: torch.Tensor | None = None, dq: torch.Tensor | None = None,
                          dk: torch.Tensor | None = None):
    """(dq, dk, dq_weight, dk_weight) of :func:`qk_norm_rope` from its inputs
    and the gradients of its outputs.  ``dq`` / ``dk`` receive the result
    (dq_out / dk_out themselves for in place)."""
    dev, B, Hq, Hk, L, D, positions, stride = _qk_checks(q, k, q_weight, k_weight, inv_freq,
                                                         positions)
    if (k is None) != (dk_out is None):
        raise ValueError("dk_out and k must be given together")
    if dq_out is None:
        raise ValueError("dq_out is required")
    _heads_out("dq_out", dq_out, q)
    dq = _heads_out("dq", dq, q)
    dwq = torch.empty_like(q_weight)
    dwk = None
    if k is not None:
        _heads_out("dk_out", dk_out, k)
        dk = _heads_out("dk", dk, k)
        dwk = torch.empty_like(k_weight)
    elif dk is not None:
        raise ValueError("dk without k")
    lib = _lib.load()
    need = lib.esa_qk_norm_rope_backward_workspace_size(B, L, Hq, Hk, D)
    ws = _empty((need,), torch.uint8, dev)
    _lib.launch(lib.esa_qk_norm_rope_backward, dev, _dtype_code(q), B, L, D, _t4(q), Hq, _t4(k), Hk,
                q_weight.data_ptr(), _lib.ptr(k_weight), eps, _lib.ptr(positions), stride,
                inv_freq.data_ptr(), _t4(dq_out), _t4(dk_out), _t4(dq), _t4(dk), dwq.data_ptr(),
                _lib.ptr(dwk), ws.data_ptr(), need)
    return dq, dk, dwq, dwk


# ---------------------------------------------------------------------------
# Rows in 8 bits
# ---------------------------------------------------------------------------
PACK_FORMATS = {"int8": 0, "e4m3": 1}
PACK_GROUP = 128


@dataclass(eq=False)
class PackedRows:
    """Rows kept in 8 bits: ``codes`` uint8 [*shape], ``scales`` float32
    [*shape[:-1], ceil(shape[-1] / 128)], one scale per 128 elements;
    ``dtype`` is the type of the rows they were made from."""
    codes: torch.Tensor
    scales: torch.Tensor
    format: str
    dtype: torch.dtype

    @property
    def shape(self) -> torch.Size:
        return self.codes.shape

    def nbytes(self) -> int:
        return self.codes.numel() + 4 * self.scales.numel()


def _pack_code(format: str) -> int:
    code = PACK_FORMATS.get(format)
    if code is None:
        raise ValueError(f"unknown 8-bit format {format!r}; expected one of {sorted(PACK_FORMATS)}")
    return code


def _new_packed(shape: tuple, format: str, dtype: torch.dtype, dev) -> PackedRows:
    return PackedRows(_empty(shape, torch.uint8, dev),
                      _empty(shape[:-1] + (-(-shape[-1] // PACK_GROUP),), torch.float32, dev),
                      format, dtype)


def _check_packed(p: PackedRows) -> int:
    """The format code of a PackedRows whose parts fit together."""
    code = _pack_code(p.format)
    shape = _shape(p.codes)
    if (p.codes.dtype != torch.uint8 or p.scales.dtype != torch.float32
            or p.scales.shape != shape[:-1] + (-(-shape[-1] // PACK_GROUP),)):
        raise ValueError("PackedRows: codes must be uint8 and scales float32 "
                         "[*codes.shape[:-1], ceil(codes.shape[-1] / 128)]")
    if not p.codes.is_contiguous() or not p.scales.is_contiguous():
        raise ValueError("PackedRows: codes and scales must be contiguous")
    return code


def quantize_rows(x: torch.Tensor, format: str = "int8") -> PackedRows:
    """x [..., dim] in 8 bits, one scale per 128 elements of the last axis:
    ``int8`` (even steps of max|x| / 127 per group) or ``e4m3`` (relative
    steps, power-of-two scales).  A group with an infinity or a NaN decodes to
    NaN, and in ``int8`` the largest float32 itself to an infinity."""
    code = _pack_code(format)
    dev = _check_device(x)
    shape = _shape(x)
    n = _rows(x, shape[-1])
    dtype_code = _dtype_code(x)
    p = _new_packed(shape, format, x.dtype, dev)
    _lib.launch(_lib.load().esa_quantize_rows, dev, dtype_code, code, n, shape[-1], x.data_ptr(),
                p.codes.data_ptr(), p.scales.data_ptr())
    return p


def dequantize_rows(packed: PackedRows, dtype: torch.dtype | None = None) -> torch.Tensor:
    """The rows that the codes stand for, in ``dtype`` (default: the dtype they
    were made from)."""
    code = _check_packed(packed)
    dev = _check_device(packed.codes, packed.scales)
    x = torch.empty_like(packed.codes, dtype=dtype or packed.dtype)
    dim = x.shape[-1]
    _lib.launch(_lib.load().esa_dequantize_rows, dev, _dtype_code(x), code, _rows(x, dim), dim,
                packed.codes.data_ptr(), packed.scales.data_ptr(), x.data_ptr())
    return x


def rmsnorm_forward_packed(x: torch.Tensor, weight: torch.Tensor, eps: float,
                           residual: torch.Tensor | None = None, format: str = "int8"):
    """(h, y, rstd, packed): :func:`rmsnorm_forward` (h bit for bit, y and rstd
    within a rounding) and h in 8 bits, in one pass."""
    code = _pack_code(format)
    dev = _check_device(x, weight)
    shape = _shape(x)
    dim = shape[-1]
    n = _rows(x, dim)
    dtype_code = _dtype_code(x)
    _check_norm_weight(weight, dim, x.dtype)
    h = x
    if residual is not None:
        if residual.shape != x.shape or residual.dtype != x.dtype or residual.device != dev:
            raise ValueError("residual must match x")
        _rows(residual, dim)
        h = torch.empty_like(x)
    y = torch.empty_like(x)
    rstd = _empty(shape[:-1], torch.float32, dev)
    p = _new_packed(shape, format, x.dtype, dev)
    _lib.launch(_lib.load().esa_rmsnorm_pack_forward, dev, dtype_code, code, n, dim, x.data_ptr(),
                _lib.ptr(residual), None if residual is None else h.data_ptr(), weight.data_ptr(),
                eps, y.data_ptr(), rstd.data_ptr(), p.codes.data_ptr(), p.scales.data_ptr())
    return h, y, rstd, p


def rmsnorm_from_packed(packed: PackedRows, weight: torch.Tensor, eps: float):
    """(h, y, rstd): the rows the codes stand for, in their dtype, and their
    RMSNorm, in one pass over the codes."""
    code = _check_packed(packed)
    dev = _check_device(packed.codes, packed.scales, weight)
    shape = tuple(packed.shape)
    _check_norm_weight(weight, shape[-1], packed.dtype)
    h = torch.empty_like(packed.codes, dtype=packed.dtype)
    y = torch.empty_like(h)
    rstd = _empty(shape[:-1], torch.float32, dev)
    _lib.launch(_lib.load().esa_rmsnorm_unpack_forward, dev, _dtype_code(h), code,
                _rows(h, shape[-1]), shape[-1], packed.codes.data_ptr(), packed.scales.data_ptr(),
                weight.data_ptr(), eps, h.data_ptr(), y.data_ptr(), rstd.data_ptr())
    return h, y, rstd


def _check_norm_weight(weight: torch.Tensor, dim: int, dtype: torch.dtype) -> None:
    if weight.shape != (dim,) or weight.dtype != dtype or not weight.is_contiguous():
        raise ValueError("weight must be a contiguous [dim] tensor of the rows' dtype")


def swiglu_forward_packed(gate_up: torch.Tensor, format: str = "int8"):
    """(out, packed): :func:`swiglu_forward` (within a rounding) and gate_up in 8
    bits, in one pass.  packed has shape [..., 2, ffn]: the gate and the up half of a row
    are rows of their own."""
    code = _pack_code(format)
    dev = _check_device(gate_up)
    shape = _shape(gate_up)
    if shape[-1] % 2:
        raise ValueError("gate_up rows must hold two halves of equal width")
    ffn = shape[-1] // 2
    n = _rows(gate_up, 2 * ffn)
    dtype_code = _dtype_code(gate_up)
    out = _empty(shape[:-1] + (ffn,), gate_up.dtype, dev)
    p = _new_packed(shape[:-1] + (2, ffn), format, gate_up.dtype, dev)
    _lib.launch(_lib.load().esa_swiglu_pack_forward, dev, dtype_code, code, n, ffn,
                gate_up.data_ptr(), out.data_ptr(), p.codes.data_ptr(), p.scales.data_ptr())
    return out, p


def swiglu_backward_packed(packed: PackedRows, dout: torch.Tensor, recompute: bool = True):
    """(d gate_up, output recomputed or None) of SwiGLU at the gate and up
    values that the codes of :func:`swiglu_forward_packed` stand for."""
    code = _check_packed(packed)
    dev = _check_device(packed.codes, packed.scales, dout)
    shape = tuple(packed.shape)
    if len(shape) < 2 or shape[-2] != 2:
        raise ValueError("packed must come from swiglu_forward_packed ([..., 2, ffn])")
    ffn = shape[-1]
    lead = shape[:-2]
    if tuple(dout.shape) != lead + (ffn,) or dout.dtype != packed.dtype:
        raise ValueError("dout must be [..., ffn] in the packed rows' dtype")
    dout = dout.contiguous()
    dgu = _empty(lead + (2 * ffn,), dout.dtype, dev)
    out = torch.empty_like(dout) if recompute else None
    _lib.launch(_lib.load().esa_swiglu_unpack_backward, dev, _dtype_code(dout), code,
                _rows(dout, ffn), ffn, packed.codes.data_ptr(), packed.scales.data_ptr(),
                dout.data_ptr(), dgu.data_ptr(), _lib.ptr(out))
    return dgu, out


# ---------------------------------------------------------------------------
# Log probabilities of tokens
# ---------------------------------------------------------------------------
MAX_TOP = 32
IGNORED_TOKEN = -100


@dataclass(eq=False)
class TokenLogProbs:
    """What :func:`token_logprobs` found in rows of logits [..., vocab], all
    float32 but the ids: ``logprobs`` and ``entropy`` [...], ``stats`` [..., 2]
    (the row's maximum m and ln of the sum of exp(x - m)), ``top_ids`` int64 and
    ``top_logprobs`` [..., top_k] (None without alternatives)."""
    logprobs: torch.Tensor
    entropy: torch.Tensor
    stats: torch.Tensor
    top_ids: torch.Tensor | None
    top_logprobs: torch.Tensor | None

    @property
    def logsumexp(self) -> torch.Tensor:
        return self.stats.sum(-1)


def _logit_rows(name: str, x: torch.Tensor) -> tuple:
    """(rows, vocab, elements between rows) of [..., vocab] rows that lie evenly
    spaced in memory (contiguous, or a 2-D view such as a slice of columns)."""
    if x.dim() == 0:
        raise ValueError(f"{name} need a vocabulary axis")
    vocab = x.shape[-1]
    if vocab == 0:
        raise ValueError(f"{name} need at least one element per row")
    if x.is_contiguous():
        return x.numel() // vocab, vocab, vocab
    if x.dim() == 2 and x.stride(1) == 1 and (x.stride(0) >= vocab or x.shape[0] <= 1):
        return x.shape[0], vocab, max(x.stride(0), vocab)
    raise ValueError(f"{name} must be contiguous, or 2-D with contiguous rows")


def _score_args(logits: torch.Tensor, tokens: torch.Tensor):
    dev = _check_device(logits, tokens)
    code = _dtype_code(logits)
    n, vocab, stride = _logit_rows("logits", logits)
    if tokens.shape != logits.shape[:-1]:
        raise ValueError("tokens must be [*logits.shape[:-1]]")
    return dev, code, n, vocab, stride, _ids(tokens)


def check_top_k(top_k: int, vocab: int) -> None:
    if not 0 <= top_k <= min(MAX_TOP, vocab):
        raise ValueError(f"top_k {top_k} outside [0, {min(MAX_TOP, vocab)}]")


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top_k: int = 0) -> TokenLogProbs:
    """Log probability of one token per row of ``logits`` [..., vocab], the
    entropy of the row and, with ``top_k`` (up to 32), its most likely tokens
    with their log probabilities, in one pass over the logits: descending, equal
    ones by ascending id.  Logits of -infinity (a mask) have probability 0; a
    row with a NaN or +infinity, or of -infinity alone, gives NaN.  Token -100
    (a row to ignore) gives 0; another one outside [0, vocab) gives NaN and sets
    ``_lib.DEVERR_TOKEN_RANGE`` (``ops.device_errors``)."""
    dev, code, n, vocab, stride, tokens = _score_args(logits, tokens)
    check_top_k(top_k, vocab)
    shape = tuple(tokens.shape)
    r = TokenLogProbs(_empty(shape, torch.float32, dev), _empty(shape, torch.float32, dev),
                      _empty(shape + (2,), torch.float32, dev), None, None)
    if top_k:
        r.top_ids = _empty(shape + (top_k,), torch.int64, dev)
        r.top_logprobs = _empty(shape + (top_k,), torch.float32, dev)
    _lib.launch(_lib.load().esa_token_logprobs_forward, dev, code, tokens.element_size(), n, vocab,
                stride, logits.data_ptr(), tokens.data_ptr(), top_k, r.logprobs.data_ptr(),
                r.entropy.data_ptr(), r.stats.data_ptr(), _lib.ptr(r.top_ids),
                _lib.ptr(r.top_logprobs))
    return r


def token_logprobs_backward(logits: torch.Tensor, tokens: torch.Tensor, scores: TokenLogProbs,
                            dlogprobs: torch.Tensor | None, dentropy: torch.Tensor | None = None,
                            out: torch.Tensor | None = None) -> torch.Tensor:
    """d logits from the gradients (float32 [...]; None = zeros) of the
    ``logprobs`` and ``entropy`` that :func:`token_logprobs` gave as ``scores``
    for the same logits and tokens.  The alternatives have no gradient.  ``out``
    receives the result (``logits`` itself for in place)."""
    dev, code, n, vocab, stride, tokens = _score_args(logits, tokens)
    shape = tokens.shape
    for name, t, want in (("scores.stats", scores.stats, shape + (2,)),
                          ("scores.entropy", scores.entropy, shape),
                          ("dlogprobs", dlogprobs, shape), ("dentropy", dentropy, shape)):
        if t is not None and (t.dtype != torch.float32 or t.shape != want or t.device != dev):
            raise ValueError(f"{name} must be float32 [{', '.join(map(str, want))}] on {dev}")
    stats, entropy = scores.stats.contiguous(), scores.entropy.contiguous()
    dlogprobs = None if dlogprobs is None else dlogprobs.contiguous()
    dentropy = None if dentropy is None else dentropy.contiguous()
    if out is None:
        out = _empty(tuple(logits.shape), logits.dtype, dev)
    elif out.shape != logits.shape or out.dtype != logits.dtype or out.device != dev:
        raise ValueError("out must match logits")
    out_stride = _logit_rows("out", out)[2]
    _lib.launch(_lib.load().esa_token_logprobs_backward, dev, code, tokens.element_size(), n, vocab,
                stride, logits.data_ptr(), tokens.data_ptr(), stats.data_ptr(), entropy.data_ptr(),
                _lib.ptr(dlogprobs), _lib.ptr(dentropy), out_stride, out.data_ptr())
    return out


# ---------------------------------------------------------------------------
# Weights in 4 bits
# ---------------------------------------------------------------------------
WEIGHT4_GROUPS = (32, 64, 128)
# Rows of a 16-bit type up to which linear4 is the faster way; beyond, a product
# with the weight decoded for it.  12288 x 4096 bf16, us: 64 rows 30 (decoded 53),
# 128 rows 55 (51), 256 rows 102 (58); 4096 x 4096 in groups of 32: 64 rows 15 (20),
# 96 rows 23 (20).  float32 rows have no such number: 4096 x 4096, 64 rows 40 (104),
# 512 rows 217 (327), 8192 rows 3041 (4226).
LINEAR4_ROWS = 64
LINEAR4_MAX_ROWS = 1 << 20     # of one call


@dataclass(eq=False)
class PackedWeight4:
    """A weight [n, k] in 4 bits: ``codes`` uint8 in the order of the product,
    ``scales`` bfloat16 [ceil(n / 16), ceil(k / 128) * 128 / group, 16], ``shape`` (n, k) and
    ``dtype`` those of the weight it was made from."""
    codes: torch.Tensor
    scales: torch.Tensor
    shape: tuple
    group: int
    dtype: torch.dtype

    def nbytes(self) -> int:
        return self.codes.numel() + 2 * self.scales.numel()


def quantize_weight4(weight: torch.Tensor, group: int = 128) -> PackedWeight4:
    """``weight`` [n, k] (a projection's, rows of outputs) in 4 bits: even steps
    of max|w| / 7 within ``group`` (32, 64 or 128) consecutive inputs of a row,
    the step a bfloat16.  A group with an infinity or a NaN decodes to NaN; the
    largest bfloat16 decodes to 1022 * 2^118, an infinity in bfloat16."""
    dev = _check_device(weight)
    if weight.dim() != 2:
        raise ValueError("weight must be [n, k]")
    n, k = weight.shape
    _rows(weight, k)
    if n == 0:
        raise ValueError("weight needs at least one row")
    if group not in WEIGHT4_GROUPS:
        raise ValueError(f"group must be one of {WEIGHT4_GROUPS}")
    code = _dtype_code(weight)
    lib = _lib.load()
    p = PackedWeight4(_empty((lib.esa_weight4_codes_size(n, k),), torch.uint8, dev),
                      _empty((-(-n // 16), -(-k // 128) * (128 // group), 16), torch.bfloat16, dev), (n, k), group,
                      weight.dtype)
    _lib.launch(lib.esa_quantize_weight4, dev, code, n, k, group, weight.data_ptr(),
                p.codes.data_ptr(), p.scales.data_ptr())
    return p


def _check_weight4(p: PackedWeight4) -> tuple:
    n, k = p.shape
    if (p.group not in WEIGHT4_GROUPS or p.codes.dtype != torch.uint8
            or p.codes.numel() != -(-n // 16) * -(-k // 128) * 1024
            or p.scales.dtype != torch.bfloat16
            or p.scales.shape != (-(-n // 16), -(-k // 128) * (128 // p.group), 16)):
        raise ValueError("PackedWeight4: codes, scales, shape and group do not fit together")
    if not p.codes.is_contiguous() or not p.scales.is_contiguous():
        raise ValueError("PackedWeight4: codes and scales must be contiguous")
    return n, k


def dequantize_weight4(packed: PackedWeight4, dtype: torch.dtype | None = None) -> torch.Tensor:
    """The weight [n, k] that the codes stand for, in ``dtype`` (default: the
    dtype it was made from)."""
    n, k = _check_weight4(packed)
    dev = _check_device(packed.codes, packed.scales)
    w = _empty((n, k), dtype or packed.dtype, dev)
    _lib.launch(_lib.load().esa_dequantize_weight4, dev, _dtype_code(w), n, k, packed.group,
                packed.codes.data_ptr(), packed.scales.data_ptr(), w.data_ptr())
    return w


def linear4(x: torch.Tensor, packed: PackedWeight4) -> torch.Tensor:
    """x [..., k] times the transposed weight: [..., n].  Exact products of x and
    the codes, float32 sums (of a group before its scale is taken: |x| up to 2^118),
    rounded once.  Made for few rows (decoding: 16-bit types up to
    ``LINEAR4_ROWS``); it takes ``LINEAR4_MAX_ROWS``."""
    n, k = _check_weight4(packed)
    dev = _check_device(x, packed.codes, packed.scales)
    shape = _shape(x)
    rows = _rows(x, k)
    code = _dtype_code(x)
    y = _empty(shape[:-1] + (n,), x.dtype, dev)
    _lib.launch(_lib.load().esa_linear4, dev, code, rows, n, k, packed.group, x.data_ptr(),
                packed.codes.data_ptr(), packed.scales.data_ptr(), y.data_ptr())
    return y
