"""GPU: keys and values cached in 4 bits and elastic attention over them, against
plain formulas in float64.

Codes and scales are exact, a value (4 bits times a bfloat16) is exact in float32:
rows written and read back are compared for equality.

Attention, u = 2^-24, per (row, head) with scores s_k, weights p_k, values v_k:
  scores   the query in fixed point is off by 2^-30 of its largest element at each
           element; D / 32 groups' sums, products with scales and units in float32:
           ds = scale (2^-30 max|q| sum|k| + (D / 32 + 8) u sum|q k|)
  weights  relative 2 ds (their own and the normaliser's) and some 12 u (exp2, the
           corrections of an online softmax, the normaliser's chain of w / 32 + 12)
  output   a weight times a scale in fixed point: off by up to 2^-16 (float32: 2^-31)
           of the largest of its 32 slots and all groups, times a code of up to 7
"""
import math

import pytest
import torch

from oracle import pattern

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def esa():
    import elastic_sparse_attention_b200 as mod
    return mod


def decoded(x):
    g = x.double().unflatten(-1, (-1, 32))
    top = g.abs().amax(-1, keepdim=True)
    s = (top.float() / torch.full_like(top, 7.0).float()).bfloat16().double().clamp_min(2.0 ** -126)
    v = torch.where(g.isfinite().all(-1, keepdim=True), torch.round(g / s) * s, math.nan)
    return v.flatten(-2)


def scales_of(x):
    top = x.double().unflatten(-1, (-1, 32)).abs().amax(-1)
    return (top.float() / torch.full_like(top, 7.0).float()).bfloat16().double().clamp_min(2.0 ** -126)


def head_rows(shape, g, dtype):
    x = torch.randn(shape, generator=g)
    x = x * torch.where(torch.rand(shape[-1:], generator=g) < 0.05, 8.0, 1.0)
    return x.to(DEV, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("B,H,S,L", [(1, 1, 1, 1), (2, 3, 50, 7), (3, 8, 40, 33), (1, 2, 700, 700)])
def test_write_and_read(esa, dtype, D, B, H, S, L):
    g = torch.Generator().manual_seed(D + S)
    cache = esa.PackedKVCache(B, H, S, D, device=DEV)
    first_k, first_v = head_rows((B, H, S, D), g, dtype), head_rows((B, H, S, D), g, dtype)
    cache.write(first_k, first_v, 0)
    # parts of a fused projection: [B, L, 3 H, D]
    qkv = head_rows((B, L, 3 * H, D), g, dtype)
    k, v = qkv[:, :, H:2 * H].transpose(1, 2), qkv[:, :, 2 * H:].transpose(1, 2)
    start = torch.randint(0, S - L + 1, (B,), generator=g)
    counts = torch.randint(0, L + 1, (B,), generator=g)
    counts[0] = L
    cache.write(k, v, start.to(DEV), counts.to(DEV))
    want_k, want_v = decoded(first_k), decoded(first_v)
    for b in range(B):
        s, n = int(start[b]), int(counts[b])
        want_k[b, :, s:s + n] = decoded(k[b, :, :n])
        want_v[b, :, s:s + n] = decoded(v[b, :, :n])
    for out in DTYPES:
        rk, rv = cache.read(0, S, out)
        assert rk.dtype == out
        assert torch.equal(rk, want_k.float().to(out)) and torch.equal(rv, want_v.float().to(out))
    rk, rv = cache.read(start.to(DEV), L, torch.float32)
    for b in range(B):
        s = int(start[b])
        assert torch.equal(rk[b].double(), want_k[b, :, s:s + L])
        assert torch.equal(rv[b].double(), want_v[b, :, s:s + L])
    assert esa.ops.device_errors() == 0


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", DTYPES)
def test_ties_extremes_and_fresh_rows(esa, D, dtype):
    g = torch.Generator().manual_seed(D)
    k = torch.randint(-14, 15, (1, 2, 60, D), generator=g) / 2.0
    k[..., ::32] = 7.0
    k = (k * 2.0 ** torch.randint(-8, 9, (1, 2, 60, 1), generator=g).float()).to(DEV, dtype)
    v = head_rows((1, 2, 60, D), g, dtype)
    v[0, 0, 3, 5] = math.nan
    v[0, 0, 4, 40] = math.inf
    v[0, 1, 5] = 0
    v[0, 1, 6] = torch.finfo(dtype).max
    v[0, 1, 7] = torch.finfo(dtype).smallest_normal
    cache = esa.PackedKVCache(1, 2, 80, D, device=DEV)
    cache.write(k, v, 10)
    rk, rv = cache.read(0, 80, torch.float32)
    assert not rk[:, :, :10].any() and not rv[:, :, 70:].any()          # never written: zeros
    assert torch.equal(rk[:, :, 10:70].double(), decoded(k))
    want = decoded(v)
    assert torch.equal(rv[:, :, 10:70].isnan(), want.isnan())
    assert torch.equal(rv[:, :, 10:70].double().nan_to_num(9.0), want.nan_to_num(9.0))
    assert torch.isfinite(rv[0, 1]).all()


def test_rows_outside_the_cache(esa):
    bit = esa._lib.DEVERR_KV_RANGE
    cache = esa.PackedKVCache(4, 1, 10, 64, device=DEV)
    old = torch.randn(4, 1, 10, 64, device=DEV)
    cache.write(old, old, 0)
    kept = decoded(old)
    esa.ops.device_errors()
    new = torch.randn(4, 1, 6, 64, device=DEV)
    start = torch.tensor([7, -3, 1 << 60, -(1 << 62)], device=DEV)
    cache.write(new, new, start)
    assert esa.ops.device_errors() == bit
    kept[0, :, 7:] = decoded(new)[0, :, :3]
    kept[1, :, :3] = decoded(new)[1, :, 3:]
    assert torch.equal(cache.read(0, 10, torch.float32)[0].double(), kept)
    assert esa.ops.device_errors() == 0
    r = cache.read(start, 6, torch.float32)[1]
    assert esa.ops.device_errors() == bit
    assert torch.equal(r[0, :, :3].double(), kept[0, :, 7:]) and not r[0, :, 3:].any()
    assert not r[1, :, :3].any() and torch.equal(r[1, :, 3:].double(), kept[1, :, :3])
    assert not r[2:].any()
    # counts below zero and beyond the rows; padding beyond the cache is no error
    cache.write(new, new, 8, torch.tensor([2, -5, 0, 1], device=DEV))
    assert esa.ops.device_errors() == 0
    kept[0, :, 8:] = decoded(new)[0, :, :2]
    kept[3, :, 8:9] = decoded(new)[3, :, :1]
    assert torch.equal(cache.read(0, 10, torch.float32)[0].double(), kept)
    cache.write(new, new, 4, torch.tensor([99, 0, 0, 0], device=DEV))
    assert esa.ops.device_errors() == 0
    kept[0, :, 4:] = decoded(new)[0]
    assert torch.equal(cache.read(0, 10, torch.float32)[0].double(), kept)


def attend64(q, k, v, sk, sv, spec, scale, start, counts):
    """(o, lse, slack of o, slack of lse) in float64: k, v decoded rows [B, Hkv, S, D],
    sv their values' scales."""
    B, Hq, L, D = q.shape
    G = Hq // k.shape[1]
    vfix = 2.0 ** -31 if q.dtype == torch.float32 else 2.0 ** -16
    w = spec.attention_length
    o = torch.zeros(B, Hq, L, D, dtype=torch.float64, device=q.device)
    lse = torch.full((B, Hq, L), -math.inf, dtype=torch.float64, device=q.device)
    so, sl = torch.zeros_like(o), torch.zeros_like(lse)
    for b in range(B):
        n = int(counts[b])
        if n == 0:
            continue
        idx, mask = pattern.elastic_indices(int(start[b]) + torch.arange(n).numpy(),
                                            spec.pattern_heads or Hq, w, spec.layer_idx,
                                            spec.num_hidden_layers)
        idx = torch.from_numpy(idx).to(q.device)[spec.head_offset:spec.head_offset + Hq]
        mask = torch.from_numpy(mask).to(q.device)[spec.head_offset:spec.head_offset + Hq].bool()
        for h in range(Hq):
            kk, vv = k[b, h // G][idx[h]], v[b, h // G][idx[h]]           # [n, w, D]
            qq = q[b, h, :n].double()
            s = (qq[:, None] * kk).sum(-1) * scale
            s = s.masked_fill(~mask[h], -math.inf)
            lse[b, h, :n] = torch.logsumexp(s, -1) / math.log(2)
            p = torch.softmax(s, -1)
            vv = torch.where(mask[h][..., None], vv, 0.0)
            o[b, h, :n] = (p[..., None] * vv).sum(1)
            ds = scale * (2.0 ** -30 * qq.abs().amax(-1)[:, None] * kk.abs().sum(-1)
                          + (D / 32 + 8) * U * (qq[:, None] * kk).abs().sum(-1))
            ds = torch.where(mask[h], ds, 0.0).amax(-1)
            rel = 2 * ds + (12 + w / 32 + 12) * U
            ps = (p[..., None] * torch.where(mask[h][..., None], sv[b, h // G][idx[h]], 0.0))
            so[b, h, :n] = (rel[:, None] * (p[..., None] * vv.abs()).sum(1)
                            + 7 * w * vfix * ps.amax((-1, -2))[:, None])
            sl[b, h, :n] = (1.5 * (ds + (12 + w / 32 + 12) * U)
                            + 3 * U * (lse[b, h, :n].abs() + s.masked_fill(~mask[h], 0).abs().amax(-1)))
    return o, lse, so, sl


def compare(esa, q, cache, spec, scale, start, counts, k, v, got=None):
    B, Hq, L, D = q.shape
    n = torch.full((B,), L) if counts is None else counts.clamp(0, L)
    o, lse = got or esa.ops.forward_packed(q, cache, spec, scale, start.to(DEV),
                                           None if counts is None else counts.to(DEV))
    want, wl, so, sl = attend64(q, decoded(k), decoded(v), scales_of(k), scales_of(v), spec, scale,
                                start, n)
    half = torch.finfo(q.dtype).eps / 2
    bound = half * (want.abs() + so) + so + (2.0 ** -25 if q.dtype == torch.float16 else 2.0 ** -140)
    bad = ~((o.double() - want).abs() <= bound)
    assert o.dtype == q.dtype and not bad.any(), (int(bad.sum()), float((o.double() - want).abs().max()))
    for b in range(B):
        m = int(n[b])
        assert ((lse[b, :, :m].double() - wl[b, :, :m]).abs() <= sl[b, :, :m]).all()
        assert not o[b, :, m:].any() and (lse[b, :, m:] == -math.inf).all()      # padding


def filled(esa, B, Hkv, S, D, dtype, g):
    k, v = head_rows((B, Hkv, S, D), g, dtype), head_rows((B, Hkv, S, D), g, dtype)
    cache = esa.PackedKVCache(B, Hkv, S, D, device=DEV)
    cache.write(k, v, 0)
    return cache, k, v


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("B,Hq,Hkv,S,L,w,layer,layers", [
    (1, 1, 1, 1, 1, 1, 0, 1), (1, 2, 1, 40, 40, 16, 1, 4), (2, 4, 4, 100, 5, 5, 3, 4),
    (3, 6, 2, 300, 33, 33, 0, 3), (1, 8, 2, 900, 260, 64, 2, 4), (2, 3, 1, 500, 70, 100, 3, 4),
    (1, 4, 2, 2000, 9, 300, 1, 2), (5, 8, 8, 260, 1, 64, 4, 8), (1, 2, 2, 4000, 3, 2048, 1, 3),
    (1, 32, 8, 700, 150, 32, 5, 8)])
def test_attention(esa, dtype, D, B, Hq, Hkv, S, L, w, layer, layers):
    g = torch.Generator().manual_seed(D + S + w)
    cache, k, v = filled(esa, B, Hkv, S, D, dtype, g)
    q = head_rows((B, L, Hq, D), g, dtype).transpose(1, 2)
    start = torch.randint(0, S - L + 1, (B,), generator=g)
    start[0] = 0
    spec = esa.PatternSpec(layer, layers, w)
    compare(esa, q, cache, spec, D ** -0.5, start, None, k, v)
    counts = torch.randint(0, L + 1, (B,), generator=g)
    counts[-1] = 0 if B > 1 else L
    compare(esa, q, cache, spec, D ** -0.5, start, counts, k, v)
    assert esa.ops.device_errors() == 0


def test_many_pairs(esa):
    """As many rows that warps take several pairs one after the other, an odd number."""
    g = torch.Generator().manual_seed(9)
    cache, k, v = filled(esa, 1, 2, 3000, 64, torch.bfloat16, g)
    q = head_rows((1, 2999, 6, 64), g, torch.bfloat16).transpose(1, 2)
    compare(esa, q, cache, esa.PatternSpec(2, 4, 40), 0.125, torch.tensor([1]),
            torch.tensor([2991]), k, v)


def test_the_16_bit_attention_of_the_decoded_rows(esa):
    """ops.forward over the rows that the cache stands for, at the same positions."""
    g = torch.Generator().manual_seed(2)
    cache, k, v = filled(esa, 2, 2, 600, 128, torch.bfloat16, g)
    q = head_rows((2, 50, 8, 128), g, torch.bfloat16).transpose(1, 2)
    dk, dv = cache.read(0, 600, torch.bfloat16)
    for layer in range(4):
        spec = esa.PatternSpec(layer, 4, 64)
        o, lse = esa.ops.forward_packed(q, cache, spec, 128 ** -0.5, 500)
        rows = torch.arange(500, 550, device=DEV)
        ro, rl = esa.ops.forward(q, dk, dv, spec, 128 ** -0.5, rows=rows)
        # The rows in bfloat16 are the decoded ones but for half a step, 2^-8, of each
        # element (8 significant bits).  So a score moves by ds <= scale (2^-8 + 2 D u)
        # sum|q k| (both sides' float32 sums in the second term), a weight by the factor
        # exp(2 ds) at most; the values by 2^-8; both outputs are rounded (2^-8 each), and
        # the cache's weights are on a grid of 2^-16 of the largest weight and scale,
        # times codes of up to 7.
        k64, v64, sv = decoded(k), decoded(v), scales_of(v)
        idx, mask = pattern.elastic_indices(range(500, 550), 8, 64, layer, 4)
        idx, mask = torch.from_numpy(idx).to(DEV), torch.from_numpy(mask).to(DEV).bool()
        for b in range(2):
            for h in range(8):
                kk, vv = k64[b, h // 4][idx[h]], v64[b, h // 4][idx[h]]
                each = q[b, h].double()[:, None] * kk * 128 ** -0.5
                ds = (2.0 ** -8 + 256 * U) * each.abs().sum(-1).masked_fill(~mask[h], 0).amax(-1)
                p = torch.softmax(each.sum(-1).masked_fill(~mask[h], -math.inf), -1)[..., None]
                grid = 7 * 64 * 2.0 ** -16 * (p * sv[b, h // 4][idx[h]]).amax((1, 2))
                mag = (p * vv.abs()).sum(1)
                bound = ((torch.expm1(2 * ds) + 2.0 ** -8 * torch.exp(2 * ds))[:, None] * mag
                         + 2.0 ** -7 * (mag * torch.exp(2 * ds)[:, None]) + grid[:, None])
                assert ((o[b, h].double() - ro[b, h].double()).abs() <= bound).all()
                assert ((lse[b, h].double() - rl[b, h].double()).abs()
                        <= ds / math.log(2) + 64 * U * (1 + rl[b, h].abs())).all()


def test_head_subset(esa):
    g = torch.Generator().manual_seed(4)
    cache, k, v = filled(esa, 1, 4, 400, 64, torch.float32, g)
    q = head_rows((1, 30, 8, 64), g, torch.float32).transpose(1, 2)
    spec = esa.PatternSpec(1, 3, 20)
    o, lse = esa.ops.forward_packed(q, cache, spec, 0.1, 350)
    part = esa.PackedKVCache(1, 2, 400, 64, device=DEV)
    part.write(k[:, 2:], v[:, 2:], 0)
    po, pl = esa.ops.forward_packed(q[:, 4:], part, spec.heads(8, 4), 0.1, 350)
    assert torch.equal(po, o[:, 4:]) and torch.equal(pl, lse[:, 4:])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_what_is_not_attended_to_does_not_matter(esa, dtype, D):
    """NaNs in rows beyond the query's position and between the pattern's keys; a NaN
    among the attended values reaches its own 32 elements only, one among the keys the
    whole row."""
    g = torch.Generator().manual_seed(D)
    S, w, pos = 500, 24, 300
    cache, k, v = filled(esa, 1, 1, S, D, dtype, g)
    spec = esa.PatternSpec(1, 3, w)
    idx, mask = pattern.elastic_indices([pos], 2, w, 1, 3)
    used = torch.zeros(S, dtype=torch.bool)
    used[torch.from_numpy(idx[mask.astype(bool)])] = True
    q = head_rows((1, 1, 2, D), g, dtype).transpose(1, 2)
    clean, cl = esa.ops.forward_packed(q, cache, spec, 0.1, pos)
    bad_k, bad_v = k.clone(), v.clone()
    bad_k[:, :, ~used] = math.nan
    bad_v[:, :, ~used] = math.inf
    cache.write(bad_k, bad_v, 0)
    o, lse = esa.ops.forward_packed(q, cache, spec, 0.1, pos)
    assert torch.equal(o, clean) and torch.equal(lse, cl)
    one = int(idx[0][0][w // 2])                       # a key of head 0
    bad_v[0, 0, one, 37] = math.nan
    cache.write(bad_k, bad_v, 0)
    o, lse = esa.ops.forward_packed(q, cache, spec, 0.1, pos)
    assert o[0, 0, 0, 32:64].isnan().all() and torch.equal(lse, cl)
    keep = torch.ones(D, dtype=torch.bool, device=DEV)
    keep[32:64] = False
    # (the other groups' weights are cut on another grid without that group's scale)
    assert (o[0, 0, 0, keep].float() - clean[0, 0, 0, keep].float()).abs().max() <= \
        2.0 ** -7 * clean.float().abs().max()
    bad_v[0, 0, one, 37] = 0
    bad_k[0, 0, one, 3] = math.nan
    cache.write(bad_k, bad_v, 0)
    o, lse = esa.ops.forward_packed(q, cache, spec, 0.1, pos)
    assert o[0, 0].isnan().all() and lse[0, 0].isnan().all()


def test_queries_outside_the_cache(esa):
    bit = esa._lib.DEVERR_QUERY_RANGE
    g = torch.Generator().manual_seed(6)
    cache, k, v = filled(esa, 3, 1, 50, 64, torch.float32, g)
    q = head_rows((3, 4, 2, 64), g, torch.float32).transpose(1, 2)
    spec = esa.PatternSpec(1, 2, 8)
    esa.ops.device_errors()
    start = torch.tensor([48, -2, 1 << 61])
    o, lse = esa.ops.forward_packed(q, cache, spec, 0.1, start.to(DEV))
    assert esa.ops.device_errors() == bit
    assert not o[0, :, 2:].any() and (lse[0, :, 2:] == -math.inf).all()
    assert not o[1:].any() and (lse[1:] == -math.inf).all()
    whole, _ = esa.ops.forward_packed(q[:, :, :2].contiguous(), cache, spec, 0.1, 48)
    assert torch.equal(o[0, :, :2], whole[0])
    assert esa.ops.device_errors() == 0
    nan_q = q.clone()
    nan_q[0, 0, 0, 5] = math.inf
    o, lse = esa.ops.forward_packed(nan_q, cache, spec, 0.1, 40)
    assert o[0, 0, 0].isnan().all() and torch.isfinite(o[0, 1]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_query_magnitudes(esa, dtype):
    """Tiny, large and zero queries: fixed point follows the largest element."""
    g = torch.Generator().manual_seed(8)
    cache, k, v = filled(esa, 1, 1, 200, 64, dtype, g)
    q = head_rows((1, 6, 1, 64), g, dtype)
    q[0, 0] *= 1e-4
    q[0, 1] *= 1e3
    q[0, 2] = 0
    q[0, 3, 0, 5] = 3000.0
    q = q.transpose(1, 2)
    compare(esa, q, cache, esa.PatternSpec(1, 2, 30), 0.01, torch.tensor([190]), None, k, v)


def test_offsets_beyond_32_bits(esa):
    """A cache of more than 2^32 bytes of codes."""
    B, H, S, D = 1, 3, 1 << 23, 256
    cache = esa.PackedKVCache(B, H, S, D, device=DEV)
    g = torch.Generator().manual_seed(1)
    L = 300
    k, v = head_rows((B, H, L, D), g, torch.bfloat16), head_rows((B, H, L, D), g, torch.bfloat16)
    cache.write(k, v, S - L)
    rk, rv = cache.read(S - L, L, torch.float32)
    assert torch.equal(rk.double(), decoded(k)) and torch.equal(rv.double(), decoded(v))
    # the window layer's keys are the last w rows
    q = head_rows((B, 2, H, D), g, torch.bfloat16).transpose(1, 2)
    o, _ = esa.ops.forward_packed(q, cache, esa.PatternSpec(0, 2, 64), 0.05, S - 2)
    small = esa.PackedKVCache(B, H, L, D, device=DEV)
    small.write(k, v, 0)
    so, _ = esa.ops.forward_packed(q, small, esa.PatternSpec(0, 2, 64), 0.05, L - 2)
    assert torch.equal(o, so)


def test_captured_with_changing_lengths(esa):
    """Write and attend captured once; replays read the tensors' new values."""
    g = torch.Generator().manual_seed(3)
    B, H, S, D = 3, 2, 200, 128
    cache, k, v = filled(esa, B, H, S, D, torch.bfloat16, g)
    other, _, _ = filled(esa, B, H, S, D, torch.bfloat16, torch.Generator().manual_seed(3))
    spec = esa.PatternSpec(1, 3, 32)
    nk, nv = (head_rows((B, H, 2, D), g, torch.bfloat16) for _ in range(2))
    q = head_rows((B, 4, 2, D), g, torch.bfloat16)
    start = torch.tensor([5, 50, 100], device=DEV)
    counts = torch.tensor([2, 1, 0], device=DEV)

    def call(c):
        c.write(nk, nv, start, counts)
        return esa.ops.forward_packed(q, c, spec, 0.1, start, counts)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call(cache)
        call(other)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, lse = call(cache)
    for step in range(4):
        start.copy_(torch.tensor([5 + 2 * step, 50 + step, 100 + step]))
        counts.copy_(torch.tensor([2, step % 3, 1]))
        nk.copy_(head_rows((B, H, 2, D), g, torch.bfloat16))
        graph.replay()
        wo, wl = call(other)
        assert torch.equal(o, wo) and torch.equal(lse, wl)
        assert torch.equal(cache.codes, other.codes) and torch.equal(cache.scales, other.scales)


def test_two_streams_at_once(esa):
    g = torch.Generator().manual_seed(7)
    parts = [filled(esa, 1, 4, 3000, 128, torch.bfloat16, g) for _ in range(2)]
    qs = [head_rows((1, 400, 16, 128), g, torch.bfloat16).transpose(1, 2) for _ in range(2)]
    spec = esa.PatternSpec(2, 4, 64)
    wants = [esa.ops.forward_packed(q, p[0], spec, 0.1, 2600) for q, p in zip(qs, parts)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(esa.ops.forward_packed(qs[i], parts[i][0], spec, 0.1, 2600))
    torch.cuda.synchronize()
    for want, got in zip(wants, outs):
        for o, lse in got:
            assert torch.equal(o, want[0]) and torch.equal(lse, want[1])


def test_refusals(esa):
    cache = esa.PackedKVCache(2, 2, 20, 64, device=DEV)
    x = torch.zeros(2, 2, 3, 64, device=DEV)
    q = torch.zeros(2, 4, 3, 64, device=DEV)
    spec = esa.PatternSpec(0, 2, 8)
    fwd = esa.ops.forward_packed
    for bad in (x[:1], x[:, :1], x[..., :32], x[0]):
        with pytest.raises(ValueError):
            cache.write(bad, bad, 0)
    with pytest.raises(ValueError):
        cache.write(x, x[:, :, :2], 0)
    with pytest.raises(TypeError):
        cache.write(x, x.half(), 0)
    with pytest.raises(TypeError):
        cache.write(x.double(), x.double(), 0)
    with pytest.raises(ValueError):
        cache.write(x.transpose(2, 3).contiguous().transpose(2, 3), x, 0)     # strided elements
    for start in (-1, torch.zeros(3, dtype=torch.int64), torch.zeros((), dtype=torch.int64)):
        with pytest.raises(ValueError, match="start"):
            cache.write(x, x, start)
        with pytest.raises(ValueError, match="start"):
            fwd(q, cache, spec, 0.1, start)
    with pytest.raises(ValueError, match="counts"):
        cache.write(x, x, 0, torch.zeros(1, dtype=torch.int64))
    with pytest.raises(TypeError):
        cache.read(0, 2, torch.float64)
    with pytest.raises(ValueError):
        cache.read(0, -1)
    with pytest.raises(ValueError, match="k_out"):
        cache.read(0, 2, k_out=x)
    for bad in (q[:1], q[:, :3], q[..., :32], q[0]):
        with pytest.raises(ValueError):
            fwd(bad, cache, spec, 0.1, 0)
    with pytest.raises(TypeError):
        fwd(q.double(), cache, spec, 0.1, 0)
    with pytest.raises(ValueError, match="out"):
        fwd(q, cache, spec, 0.1, 0, out=q[:, :2])
    with pytest.raises(esa._lib.EsaError, match="layer"):
        fwd(q, cache, esa.PatternSpec(5, 2, 8), 0.1, 0)
    with pytest.raises(esa._lib.EsaError, match="attention_length"):
        fwd(q, cache, esa.PatternSpec(0, 2, 4096), 0.1, 0)
    cache.write(x[:, :, :0], x[:, :, :0], 0)
    assert fwd(q[:, :, :0], cache, spec, 0.1, 0)[0].shape == (2, 4, 0, 64)
    assert cache.read(0, 0)[0].shape == (2, 2, 0, 64)
