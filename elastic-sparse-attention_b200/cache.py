"""Keys and values kept in 4 bits for decoding.

The reference attends to key / value tensors that its caller keeps (a cache of
16-bit rows, ``elastic_sparse_attention.py:728-765`` with ``cache_position``);
it has no cache of its own.  At a million tokens those rows are most of a
serving GPU's memory, and elastic attention reads few of them per token, so what
a smaller cache buys is context.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .layer_ops import _empty
from .ops import MAX_POSITION, _check_device, _span_args

CACHE_GROUP = 32
HEAD_DIMS = (64, 128, 256)


class PackedKVCache:
    """Key and value rows of ``batch`` sequences of up to ``max_len`` positions in
    4 bits, a bfloat16 scale per 32 elements: even steps of max|x| / 7 (4.5 bits
    an element, 144 bytes a position and head of 128 instead of 512).

    ``codes`` uint8 [batch, num_kv_heads, max_len, 2, head_dim / 2] (keys, then
    values; the order within a row is the kernels') and ``scales`` bfloat16
    [batch, num_kv_heads, max_len, 2, head_dim / 32] start at zero, which
    stands for zero rows.

    The rows of a call are positions ``start[b] + l``: ``start`` is an int or an
    int64 [batch] tensor, ``counts`` [batch] the number of rows each sequence
    brings (default: all; the rest of them is padding).  Nothing is read back to
    the host, so calls can be captured into a CUDA graph whose replays read the
    tensors' new values."""

    def __init__(self, batch: int, num_kv_heads: int, max_len: int, head_dim: int, device=None):
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"head_dim {head_dim} is not one of {HEAD_DIMS}")
        if batch < 0 or num_kv_heads < 1 or not 1 <= max_len <= MAX_POSITION:
            raise ValueError(f"bad cache shape: batch {batch}, num_kv_heads {num_kv_heads}, "
                             f"max_len {max_len}")
        device = torch.device("cuda" if device is None else device)
        if device.type == "cuda" and device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        shape = (batch, num_kv_heads, max_len, 2)
        self._codes = torch.zeros(shape + (head_dim // 2,), dtype=torch.uint8, device=device)
        self._scales = torch.zeros(shape + (head_dim // CACHE_GROUP,), dtype=torch.bfloat16,
                                   device=device)
        self.batch, self.num_kv_heads, self.max_len = batch, num_kv_heads, max_len
        self.head_dim = head_dim
        # the C ABI's view of the cache, whose tensors stay where they are
        self.struct = _lib.EsaCache4(self._codes.data_ptr(), self._scales.data_ptr(), batch,
                                     num_kv_heads, head_dim, 0, max_len)

    @property
    def codes(self) -> torch.Tensor:
        return self._codes

    @property
    def scales(self) -> torch.Tensor:
        return self._scales

    @property
    def device(self) -> torch.device:
        return self._codes.device

    def nbytes(self) -> int:
        return self.codes.numel() + 2 * self.scales.numel()

    def _check_rows(self, name: str, x: torch.Tensor, length: int) -> None:
        want = (self.batch, self.num_kv_heads, length, self.head_dim)
        if tuple(x.shape) != want:
            raise ValueError(f"{name} must be {list(want)}, got {list(x.shape)}")

    def write(self, k: torch.Tensor, v: torch.Tensor, start, counts=None) -> None:
        """Rows of k and v [batch, num_kv_heads, L, head_dim] (strided views with a
        contiguous last axis) into positions start + l.  Positions beyond the
        cache are left out and set ``_lib.DEVERR_KV_RANGE``
        (``ops.device_errors``); all others keep what they held."""
        dev = _check_device(k, v, self.codes)
        if k.dim() != 4:
            raise ValueError("k must be [batch, num_kv_heads, L, head_dim]")
        L = k.shape[2]
        self._check_rows("k", k, L)
        self._check_rows("v", v, L)
        if v.dtype != k.dtype or k.dtype not in _lib.DTYPES:
            raise TypeError(f"k and v must share one of {sorted(map(str, _lib.DTYPES))}")
        start, start0, counts = _span_args(self.batch, start, counts, dev)
        _lib.launch(_lib.load().esa_cache4_write, dev, _lib.DTYPES[k.dtype],
                    ctypes.byref(self.struct), L, _lib.tensor4(k), _lib.tensor4(v),
                    _lib.ptr(start), start0, _lib.ptr(counts))

    def read(self, start, length: int, dtype: torch.dtype = torch.bfloat16,
             k_out: torch.Tensor | None = None, v_out: torch.Tensor | None = None):
        """(k, v) [batch, num_kv_heads, length, head_dim]: what the codes of
        positions start + l stand for, e.g. a prefix for the 16-bit attention.
        Positions beyond the cache give zeros and set
        ``_lib.DEVERR_KV_RANGE``."""
        dev = _check_device(self.codes)
        if dtype not in _lib.DTYPES:
            raise TypeError(f"unsupported dtype {dtype}")
        if length < 0:
            raise ValueError(f"length {length} is negative")
        shape = (self.batch, self.num_kv_heads, length, self.head_dim)
        out = []
        for name, t in (("k_out", k_out), ("v_out", v_out)):
            if t is None:
                t = _empty(shape, dtype, dev)
            elif tuple(t.shape) != shape or t.dtype != dtype or t.device != dev:
                raise ValueError(f"{name} must be {list(shape)} in {dtype} on {dev}")
            out.append(t)
        start, start0, _ = _span_args(self.batch, start, None, dev)
        _lib.launch(_lib.load().esa_cache4_read, dev, _lib.DTYPES[dtype],
                    ctypes.byref(self.struct), length, _lib.tensor4(out[0]),
                    _lib.tensor4(out[1]), _lib.ptr(start), start0)
        return tuple(out)
