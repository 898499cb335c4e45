"""GPU: the 4-bit key / value cache and the attention over it at the ends of their
range: calls of more rows than the cache has positions, values whose groups differ
in size.

Attention, u = 2^-24: the bounds of test_gpu_cache4.py, but a weight times a scale is
off by up to 2^-16 (float32: 2^-31) of the largest of its 32 slots within its own
group, times a code of up to 7.  Groups are other output elements, so what one holds
does not touch another.
"""
import math

import pytest
import torch

from oracle import pattern
from test_gpu_cache4 import DEV, DTYPES, U, decoded, head_rows, scales_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def esa():
    import elastic_sparse_attention_b200 as mod
    return mod


@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("S,L", [(10, 25), (10, 10), (1, 300), (70, 1000)])
def test_more_rows_than_the_cache_has_positions(esa, D, S, L):
    """Row l is position start + l, and only positions of the cache are written or
    read, however far outside the call begins."""
    starts = [0, 1, S - 1, S, S + 1, 1 << 62, -1, -(S - 1), -S, -(S + 1), -(S + 5), -(L - 1), -L,
              -(L + 1), -(L + S), -(1 << 24), -(1 << 40), -(1 << 62)]
    B = len(starts)
    g = torch.Generator().manual_seed(S + L)
    old, new = head_rows((B, 2, S, D), g, torch.float32), head_rows((B, 2, L, D), g, torch.float32)
    start = torch.tensor(starts, device=DEV)
    for counts in (None, torch.full((B,), L - L // 3)):
        n = L if counts is None else int(counts[0])
        cache = esa.PackedKVCache(B, 2, S, D, device=DEV)
        cache.write(old, old, 0)
        esa.ops.device_errors()
        cache.write(new, new, start, None if counts is None else counts.to(DEV))
        assert esa.ops.device_errors() == esa._lib.DEVERR_KV_RANGE
        want = decoded(old)
        fresh = decoded(new)
        for b, s in enumerate(starts):
            for p in range(max(s, 0), min(s + n, S)):
                want[b, :, p] = fresh[b, :, p - s]
        for t in cache.read(0, S, torch.float32):
            assert torch.equal(t.double(), want)
        out = torch.zeros(B, 2, L, D, dtype=torch.float64, device=DEV)
        for b, s in enumerate(starts):
            for p in range(max(s, 0), min(s + L, S)):
                out[b, :, p - s] = want[b, :, p]
        assert esa.ops.device_errors() == 0
        for t in cache.read(start, L, torch.float32):
            assert torch.equal(t.double(), out)
        assert esa.ops.device_errors() == esa._lib.DEVERR_KV_RANGE


def row64(q, kk, vv, sv, keep, scale, vfix):
    """(o [D], lse, slack of o, slack of lse) in float64 of one query [D] over its w
    keys and values [w, D] with the values' scales [w, D / 32]."""
    w, D = kk.shape
    kk, vv, sv = kk[keep], vv[keep], sv[keep]
    s = kk @ q * scale
    p = torch.softmax(s, 0)
    lse = torch.logsumexp(s, 0) / math.log(2)
    ds = (scale * (2.0 ** -30 * q.abs().max() * kk.abs().sum(1)
                   + (D / 32 + 8) * U * (kk * q).abs().sum(1))).max()
    chain = (12 + w / 32 + 12) * U
    grid = 7 * w * vfix * (p[:, None] * sv).amax(0).repeat_interleave(32)
    return (p @ vv, lse, (2 * ds + chain) * (p @ vv.abs()) + grid,
            1.5 * (ds + chain) + 3 * U * (lse.abs() + s.abs().max()))


def check_row(o, lse, want):
    wo, wl, so, sl = want
    bound = torch.finfo(o.dtype).eps / 2 * (wo.abs() + so) + so
    bound = bound + (2.0 ** -25 if o.dtype == torch.float16 else 2.0 ** -140)
    off = (o.double() - wo).abs()
    assert (off <= bound).all(), (int((off > bound).sum()), float((off / bound).max()))
    assert (lse.double() - wl).abs() <= sl


def fixed_point(dtype):
    return 2.0 ** -31 if dtype == torch.float32 else 2.0 ** -16


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("ratio", [64, 4096, 100000])
@pytest.mark.parametrize("L,w", [(3, 64), (3, 200), (50, 64)])
def test_values_whose_groups_differ_in_size(esa, dtype, D, ratio, L, w):
    """The groups of 32 channels of a value by turns large and `ratio` times smaller:
    each output is as exact as its own group allows."""
    g = torch.Generator().manual_seed(D + ratio)
    S, Hq, Hkv = 700, 6, 3
    gain = torch.tensor([64.0 / ratio, 64.0]).repeat(D // 64).repeat_interleave(32)
    k = head_rows((1, Hkv, S, D), g, dtype)
    v = (torch.randn(1, Hkv, S, D, generator=g) * gain).to(DEV, dtype)
    q = head_rows((1, L, Hq, D), g, dtype).transpose(1, 2)
    cache = esa.PackedKVCache(1, Hkv, S, D, device=DEV)
    cache.write(k, v, 0)
    spec = esa.PatternSpec(2, 4, w)
    start = S - L
    o, lse = esa.ops.forward_packed(q, cache, spec, D ** -0.5, start)
    dk, dv, sv = decoded(k), decoded(v), scales_of(v)
    rows = [0, L - 1] if L < 10 else range(0, L, 7)
    idx, mask = pattern.elastic_indices([start + r for r in rows], Hq, w, 2, 4)
    for h in range(Hq):
        for i, r in enumerate(rows):
            at = torch.from_numpy(idx[h, i]).to(DEV)
            keep = torch.from_numpy(mask[h, i]).to(DEV).bool()
            check_row(o[0, h, r], lse[0, h, r],
                      row64(q[0, h, r].double(), dk[0, h // 2][at], dv[0, h // 2][at],
                            sv[0, h // 2][at], keep, D ** -0.5, fixed_point(dtype)))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("L", [1, 700])
def test_a_group_does_not_touch_the_others(esa, dtype, D, L):
    """Another group's values, its NaNs among them, leave a group's outputs as they
    were, bit for bit."""
    g = torch.Generator().manual_seed(D + L)
    S, w = 900, 40
    k, v = (head_rows((1, 2, S, D), g, dtype) for _ in range(2))
    q = head_rows((1, L, 4, D), g, dtype).transpose(1, 2)
    spec = esa.PatternSpec(1, 3, w)
    cache = esa.PackedKVCache(1, 2, S, D, device=DEV)
    cache.write(k, v, 0)
    clean, cl = esa.ops.forward_packed(q, cache, spec, 0.1, S - L)
    keep = torch.ones(D, dtype=torch.bool, device=DEV)
    keep[32:64] = False
    for other in (500.0 * v[..., 32:64], 0 * v[..., 32:64], math.nan):
        changed = v.clone()
        changed[..., 32:64] = other
        cache.write(k, changed, 0)
        o, lse = esa.ops.forward_packed(q, cache, spec, 0.1, S - L)
        assert torch.equal(o[..., keep], clean[..., keep]) and torch.equal(lse, cl)
    assert o[..., 32:64].isnan().all()


def test_a_batch_of_no_sequences(esa):
    cache = esa.PackedKVCache(0, 2, 10, 64, device=DEV)
    x = torch.zeros(0, 2, 3, 64, device=DEV)
    for start in (0, torch.zeros(0, dtype=torch.int64, device=DEV)):
        cache.write(x, x, start)
        assert [t.shape for t in cache.read(start, 3)] == [(0, 2, 3, 64)] * 2
        o, lse = esa.ops.forward_packed(torch.zeros(0, 4, 3, 64, device=DEV), cache,
                                        esa.PatternSpec(1, 2, 8), 0.1, start)
        assert o.shape == (0, 4, 3, 64) and lse.shape == (0, 4, 3)
    assert esa.ops.device_errors() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layer,layers,w", [(1, 4, 64), (5, 8, 100), (3, 4, 33), (0, 4, 64)])
def test_positions_next_to_2_24(esa, dtype, layer, layers, w):
    """Strided and window layers at the end of the longest cache: only the rows of the
    definition's pattern hold anything, so that another row would show."""
    S, D, L, Hq = 1 << 24, 64, 4, 2
    g = torch.Generator().manual_seed(w)
    cache = esa.PackedKVCache(1, 1, S, D, device=DEV)
    idx, mask = pattern.elastic_indices(range(S - L, S), Hq, w, layer, layers)
    mask = mask.astype(bool)
    places = sorted(set(idx[mask].tolist()))
    assert places[-1] < S and places[0] >= 0
    k, v = (head_rows((1, 1, len(places), D), g, dtype) for _ in range(2))
    for i, p in enumerate(places):
        cache.write(k[:, :, i:i + 1], v[:, :, i:i + 1], p)
    q = head_rows((1, L, Hq, D), g, dtype).transpose(1, 2)
    o, lse = esa.ops.forward_packed(q, cache, esa.PatternSpec(layer, layers, w), D ** -0.5, S - L)
    dk, dv, sv = decoded(k)[0, 0], decoded(v)[0, 0], scales_of(v)[0, 0]
    which = {p: i for i, p in enumerate(places)}
    for h in range(Hq):
        for r in range(L):
            at = torch.tensor([which[p] for p in idx[h, r][mask[h, r]].tolist()], device=DEV)
            keep = torch.ones(len(at), dtype=torch.bool, device=DEV)
            wo, wl, so, sl = row64(q[0, h, r].double(), dk[at], dv[at], sv[at], keep, D ** -0.5,
                                   fixed_point(dtype) * w / len(at))
            check_row(o[0, h, r], lse[0, h, r], (wo, wl, so, sl))
    assert esa.ops.device_errors() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("L", [1, 600])
def test_outputs_in_place_of_the_queries(esa, dtype, L):
    """`out` may be q itself, or rows of another layout."""
    g = torch.Generator().manual_seed(L)
    k, v = (head_rows((2, 2, 900, 128), g, dtype) for _ in range(2))
    cache = esa.PackedKVCache(2, 2, 900, 128, device=DEV)
    cache.write(k, v, 0)
    q = head_rows((2, L, 8, 128), g, dtype).transpose(1, 2)
    spec = esa.PatternSpec(2, 4, 64)
    want, wl = esa.ops.forward_packed(q, cache, spec, 0.1, 300)
    rows = torch.full((2, 8, L, 256), 3.0, device=DEV, dtype=dtype)
    o, lse = esa.ops.forward_packed(q, cache, spec, 0.1, 300, out=rows[..., 64:192])
    assert torch.equal(o, want) and torch.equal(lse, wl)
    assert (rows[..., :64] == 3).all() and (rows[..., 192:] == 3).all()
    o, lse = esa.ops.forward_packed(q, cache, spec, 0.1, 300, out=q)
    assert torch.equal(q, want) and torch.equal(lse, wl)
