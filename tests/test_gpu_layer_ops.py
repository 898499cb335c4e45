"""GPU: token embedding and its gradient, per-head query / key norm with the
rotary embedding, rows in 8 bits, against plain formulas in float64.

Tolerances count roundings.  u = 2^-24 is float32's unit; a result is rounded
once to its dtype (``half_step``).  A float32 sum of m terms is off by at most
(m - 1) u times the sum of their magnitudes, whatever its order.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def check(got, want, dtype, slack, what):
    """|got - want| <= half a step of dtype at want, plus ``slack`` (the error
    of the float32 arithmetic before the rounding), which may itself move the
    rounding: half a step relative to |want| + slack."""
    assert got.dtype == dtype and got.shape == want.shape, what
    half_step = torch.finfo(dtype).eps / 2
    bound = half_step * (want.abs() + slack) + slack + TINY[dtype] / 2
    err = (got.double() - want).abs()
    bad = ~(err <= bound)
    assert not bad.any(), (what, int(bad.sum()), float((err - bound)[bad].max()),
                           float(err.max()))


@pytest.fixture(scope="module")
def lops():
    import elastic_sparse_attention_b200 as esa
    return esa.layer_ops


@pytest.fixture(scope="module")
def esa_mod():
    import elastic_sparse_attention_b200 as esa
    return esa


# ---------------------------------------------------------------------------
# embedding
# ---------------------------------------------------------------------------
def make_ids(kind, n, V, g):
    if kind == "same":
        return torch.full((n,), V // 2, dtype=torch.int64)
    if kind == "distinct":       # every token at most once where V allows, descending
        return torch.arange(n, dtype=torch.int64).flip(0) % V
    if kind == "runs":           # few tokens, long runs of different lengths
        return (torch.arange(n) // 37 * 7919 % min(V, 11)).to(torch.int64)
    u = torch.rand(n, generator=g, dtype=torch.float64)      # long-tailed
    return ((V + 1.0) ** u - 1).long().clamp(0, V - 1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,V,d,scale", [
    ((1,), 1, 8, 1.0), ((2, 0), 5, 16, 1.0), ((3, 7), 100, 24, 3.7), ((513,), 1000, 264, 16.0),
    ((2, 65), 32000, 4096, 64.0), ((1, 4097), 777, 1032, 1.0)])
def test_embedding_forward(lops, dtype, shape, V, d, scale):
    g = torch.Generator().manual_seed(V + d)
    ids = torch.randint(0, V, shape, generator=g)
    w = torch.randn(V, d, generator=g).to(DEV, dtype)
    for idt in (torch.int64, torch.int32):
        out = lops.embedding_forward(ids.to(DEV, idt), w, scale)
        want = w.double()[ids.to(DEV)] * torch.tensor(scale, dtype=torch.float32).double().item()
        check(out, want, dtype, U * want.abs(), "embedding")     # one float32 product
        if scale == 1.0:
            assert torch.equal(out, w[ids.to(DEV)])


def test_embedding_out_of_range_ids(lops, esa_mod):
    bit = esa_mod._lib.DEVERR_TOKEN_RANGE
    w = torch.randn(10, 512, device=DEV)
    esa_mod.ops.device_errors()
    ids = torch.tensor([3, -1, 10, 9, 1 << 40, -(1 << 62)], device=DEV)
    out = lops.embedding_forward(ids, w, 2.0)
    assert esa_mod.ops.device_errors() == bit
    assert torch.equal(out[[0, 3]], 2 * w[[3, 9]])
    assert not out[[1, 2, 4, 5]].any()
    for n in (6, 6000):                        # few tokens and sorted tokens
        big = ids.repeat(n // 6)
        dw = lops.embedding_backward(big, torch.ones(n, 512, device=DEV), 10)
        assert esa_mod.ops.device_errors() == bit
        want = torch.zeros(10, 512, device=DEV)
        want[3] = want[9] = n // 6
        assert torch.equal(dw, want)
    lops.embedding_forward(ids[:1], w)
    assert esa_mod.ops.device_errors() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["tail", "same", "distinct", "runs"])
@pytest.mark.parametrize("n,V,d", [
    (0, 3, 8), (1, 1, 16), (5, 700, 264), (63, 9, 8), (1023, 50, 1032), (1024, 33000, 16),
    (1025, 40, 1024), (2048, 33000, 64), (2049, 600, 256), (4096, 70000, 8), (4099, 2, 264),
    (4160, 512, 8), (9000, 70000, 24), (20001, 300000, 8),
    # the other piece lengths of wide rows
    (5000, 90, 264), (12001, 900, 264), (70001, 5000, 264),
    # around the most keys that one CTA sorts
    (2305, 70000, 8), (2559, 33000, 264), (2560, 300, 264), (2561, 33000, 264)])
def test_embedding_backward(lops, dtype, kind, n, V, d):
    g = torch.Generator().manual_seed(n + V)
    ids = make_ids(kind, n, V, g).to(DEV)
    dy = torch.randn(n, d, generator=g).to(DEV, dtype)
    scale = 1.5
    pad = int(ids[n // 2]) if n > 2 and kind in ("tail", "runs") else None
    dw = lops.embedding_backward(ids, dy, V, scale, padding_idx=pad)
    want = torch.zeros(V, d, dtype=torch.float64, device=DEV).index_add_(0, ids, dy.double())
    mag = torch.zeros(V, d, dtype=torch.float64, device=DEV).index_add_(0, ids, dy.double().abs())
    if pad is not None:
        want[pad] = 0
        mag[pad] = 0
    count = torch.bincount(ids, minlength=V).double()[:, None]
    check(dw, want * scale, dtype, count * U * mag * scale, "dweight")
    assert torch.equal(dw, lops.embedding_backward(ids.to(torch.int32), dy, V, scale,
                                                   padding_idx=pad))       # the same in every run


def test_embedding_gradient_is_the_difference_quotient(lops):
    """<dW, D> against (f(W + hD) - f(W - hD)) / 2h of f = <out, C>: f is
    linear in W, so the quotient has no truncation error (float64 formula)."""
    g = torch.Generator().manual_seed(0)
    ids = torch.randint(0, 40, (3, 500), generator=g).to(DEV)
    C = torch.randn(3, 500, 64, generator=g).to(DEV)
    W, D = (torch.randn(40, 64, generator=g, dtype=torch.float64).to(DEV) for _ in range(2))
    f = lambda w: (1.25 * w[ids] * C.double()).sum()
    quotient = (f(W + D) - f(W - D)) / 2
    dw = lops.embedding_backward(ids, C, 40, 1.25)
    terms = (dw.double() * D).abs().sum()
    # each dW entry: sums of up to ~60 terms and two roundings
    assert abs((dw.double() * D).sum() - quotient) <= 100 * U * (
        terms + (1.25 * D[ids] * C.double()).abs().sum())


# ---------------------------------------------------------------------------
# query / key norm + rotary embedding
# ---------------------------------------------------------------------------
def rotate64(x, pos, inv, sign=1.0):
    """x [B, H, L, D] float64, pos [B or 1, L]."""
    ang = pos.double()[:, None, :, None] * inv.double()
    c, s = ang.cos(), sign * ang.sin()
    a, b = x.chunk(2, -1)
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def qk_forward64(x, w, pos, inv, eps):
    x = x.double()
    rstd = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    n = x * rstd * w.double()
    a, b = n.abs().chunk(2, -1)
    return rotate64(n, pos, inv), torch.cat([a + b, a + b], -1)


# float32 error of an output of the norm and rotation, relative to |n1| + |n2|:
# sum of squares (<= 2E + log2 steps, halved by the root) 12 u, rsqrtf 4 u,
# three products and the rotation's two 5 u, cos / sin and the rounded angle
# (pi * u) 8 u: below 32 u
ROT = 32 * U


def qk_case(dtype, B, L, Hq, Hk, D, seed, far=False):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(B, L, Hq + 2 * Hk, D, generator=g)
    qkv[:, :, 0] *= 1e-3
    qkv = qkv.to(DEV, dtype)
    q = qkv[:, :, :Hq].transpose(1, 2)
    k = qkv[:, :, Hq:Hq + Hk].transpose(1, 2)
    wq, wk = ((1 + 0.3 * torch.randn(D, generator=g)).to(DEV, dtype) for _ in range(2))
    wq[0] = 0
    pos = torch.randint(0, 1 << 24 if far else 5000, (B, L), generator=g).to(DEV)
    return qkv, q, k, wq, wk, pos


QK_SHAPES = [(1, 1, 32, 8, 128), (2, 333, 4, 2, 64), (3, 5, 3, 1, 16), (1, 70, 5, 5, 32),
             (2, 40, 6, 2, 128), (1, 3, 1, 1, 64), (1, 2100, 8, 2, 128),
             # few heads, several tokens per warp: whole and partial last tasks, odd heads,
             # tasks across the batch border
             (3, 2400, 1, 1, 16), (2, 5003, 3, 1, 32), (1, 9001, 2, 1, 128), (5, 1900, 5, 2, 64),
             (1, 4800, 8, 1, 32)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,L,Hq,Hk,D", QK_SHAPES + [(2, 19, 3, 2, 256), (2, 19, 3, 2, 8)])
def test_qk_norm_rope_forward(lops, dtype, B, L, Hq, Hk, D):
    if (D == 256) == (dtype == torch.float32) and D in (8, 256):
        pytest.skip("8 is for float32, 256 for the 16-bit types")
    qkv, q, k, wq, wk, pos = qk_case(dtype, B, L, Hq, Hk, D, L + D, far=True)
    before = qkv.clone()
    inv = lops.rope_inv_freq(D, 10000.0, DEV)
    q2, k2 = lops.qk_norm_rope(q, k, wq, wk, 1e-6, inv, positions=pos)
    for got, x, w in ((q2, q, wq), (k2, k, wk)):
        want, mag = qk_forward64(x, w, pos, inv, 1e-6)
        check(got, want, dtype, ROT * mag, "norm + rotation")
    assert torch.equal(qkv, before)
    # shared positions, the default ones, no keys
    q3, _ = lops.qk_norm_rope(q, None, wq, None, 1e-6, inv, positions=pos[0])
    want, mag = qk_forward64(q, wq, pos[:1], inv, 1e-6)
    check(q3, want, dtype, ROT * mag, "shared positions")
    q4, k4 = lops.qk_norm_rope(q, k, wq, wk, 1e-6, inv)
    want, mag = qk_forward64(k, wk, torch.arange(L, device=DEV)[None], inv, 1e-6)
    check(k4, want, dtype, ROT * mag, "default positions")
    # in place: q and k rotate where they are, the values stay
    lops.qk_norm_rope(q, k, wq, wk, 1e-6, inv, positions=pos, q_out=q, k_out=k)
    assert torch.equal(q, q2) and torch.equal(k, k2)
    assert torch.equal(qkv[:, :, Hq + Hk:], before[:, :, Hq + Hk:])


def test_qk_norm_rope_far_and_negative_positions(lops):
    """The angle is exact in float64, so position 2^40 + 1 is as good as 1."""
    D = 64
    inv = lops.rope_inv_freq(D, 10000.0, DEV)
    q = torch.randn(1, 2, 6, D, generator=torch.Generator().manual_seed(1)).to(DEV)
    w = torch.ones(D, device=DEV)
    pos = torch.tensor([0, -1, -(1 << 30), (1 << 24) + 1, 1 << 31, 1 << 40], device=DEV)
    got, _ = lops.qk_norm_rope(q, None, w, None, 0.0, inv, positions=pos)
    # cos / sin of 2^40 in float64: the reference's own angle is off by 2^40 2^-53 = 2^-13;
    # both sides form the same float64 product, but differ in the reduction: compare with a
    # reduction in integers of the exact product instead
    from fractions import Fraction
    import math
    pi = Fraction(314159265358979323846264338327950288419716939937510, 10 ** 50)
    ang = torch.tensor([[float((Fraction(int(p)) * Fraction(float(f))) % (2 * pi))
                         for f in inv.cpu()] for p in pos.cpu()], dtype=torch.float64, device=DEV)
    x = q.double()
    n = x * x.square().mean(-1, keepdim=True).rsqrt()
    a, b = n.chunk(2, -1)
    want = torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()], -1)
    mag = torch.cat([a.abs() + b.abs()] * 2, -1)
    # the turns p f / 2 pi carry 2 roundings of float64: 2 pi 2^-52 |turns|
    turns = (pos.double()[:, None] * inv.double()).abs() / (2 * math.pi)
    slack = (ROT + 2 * math.pi * 2.0 ** -52 * torch.cat([turns, turns], -1)) * mag
    check(got, want, torch.float32, slack, "far positions")


def test_qk_norm_rope_zero_rows_and_specials(lops):
    D = 128
    inv = lops.rope_inv_freq(D, 10000.0, DEV)
    w = torch.ones(D, device=DEV, dtype=torch.bfloat16)
    q = torch.randn(1, 4, 3, D, device=DEV).to(torch.bfloat16)
    q[0, 1] = 0
    q[0, 2, 1, 5] = float("inf")
    q[0, 3, 2, 7] = float("nan")
    got, _ = lops.qk_norm_rope(q, None, w, None, 1e-6, inv)
    assert not got[0, 1].any()
    assert got[0, 2, 1].isnan().any() and got[0, 3, 2].isnan().all()
    clean = torch.ones(4, 3, dtype=torch.bool, device=DEV)
    clean[2, 1] = clean[3, 2] = False
    assert got[0][clean].isfinite().all()
    dq, _, dw, _ = lops.qk_norm_rope_backward(q[:, :2], None, w, None, 1e-6, inv,
                                              torch.ones_like(q[:, :2]), None)
    assert dq.isfinite().all() and dw.isfinite().all()


def qk_backward64(x, w, pos, inv, eps, dout):
    """(dx, dw) and the magnitudes that their float32 errors are relative to."""
    x, w, d = x.double(), w.double(), dout.double()
    D = x.shape[-1]
    rstd = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    xh = x * rstd
    gr = rotate64(d, pos, inv, sign=-1.0)
    a, b = d.abs().chunk(2, -1)
    gmag = torch.cat([a + b, a + b], -1)
    dx = rstd * (w * gr - xh * (xh * w * gr).mean(-1, keepdim=True))
    dxmag = rstd * (w.abs() * gmag + xh.abs() * (xh * w).abs().mul(gmag).mean(-1, keepdim=True))
    return dx, (gr * xh).sum((0, 1, 2)), dxmag, (gmag * xh.abs()).sum((0, 1, 2))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,L,Hq,Hk,D", QK_SHAPES + [(2, 19, 3, 2, 256), (2, 19, 3, 2, 8)])
def test_qk_norm_rope_backward(lops, dtype, B, L, Hq, Hk, D):
    if (D == 256) == (dtype == torch.float32) and D in (8, 256):
        pytest.skip("8 is for float32, 256 for the 16-bit types")
    qkv, q, k, wq, wk, pos = qk_case(dtype, B, L, Hq, Hk, D, L + D + 1)
    dqkv = torch.randn(qkv.shape, generator=torch.Generator().manual_seed(5)).to(DEV, dtype)
    dqo = dqkv[:, :, :Hq].transpose(1, 2)
    dko = dqkv[:, :, Hq:Hq + Hk].transpose(1, 2)
    inv = lops.rope_inv_freq(D, 10000.0, DEV)
    dq, dk, dwq, dwk = lops.qk_norm_rope_backward(q, k, wq, wk, 1e-6, inv, dqo, dko, positions=pos)
    for dx, dw, x, w, do in ((dq, dwq, q, wq, dqo), (dk, dwk, k, wk, dko)):
        want, wantw, mag, magw = qk_backward64(x, w, pos, inv, 1e-6, do)
        # the forward's 32 u, the products of the gradient 8 u, the row's mean 12 u
        check(dx, want, dtype, 64 * U * mag, "dx")
        terms = B * L * x.shape[1]
        # a sum of all rows in order and of each term's own error
        check(dw, wantw, dtype, (64 + min(terms, 4096)) * U * magw, "dweight")
    again = lops.qk_norm_rope_backward(q, k, wq, wk, 1e-6, inv, dqo, dko, positions=pos)
    assert all(torch.equal(a, b) for a, b in zip((dq, dk, dwq, dwk), again))
    # queries alone; in place on the gradients
    dq1, none, dwq1, none_w = lops.qk_norm_rope_backward(q, None, wq, None, 1e-6, inv, dqo, None,
                                                         positions=pos)
    assert none is None and none_w is None and torch.equal(dq1, dq)
    check(dwq1, qk_backward64(q, wq, pos, inv, 1e-6, dqo)[1], dtype,
          (64 + min(B * L * Hq, 4096)) * U * qk_backward64(q, wq, pos, inv, 1e-6, dqo)[3], "dwq")
    lops.qk_norm_rope_backward(q, k, wq, wk, 1e-6, inv, dqo, dko, positions=pos, dq=dqo, dk=dko)
    assert torch.equal(dqo, dq) and torch.equal(dko, dk)


def test_qk_norm_rope_gradient_is_the_difference_quotient(lops):
    g = torch.Generator().manual_seed(3)
    B, H, L, D = 1, 3, 5, 32
    inv = lops.rope_inv_freq(D, 10000.0, DEV)
    x = torch.randn(B, H, L, D, generator=g).to(DEV)
    w = (1 + 0.2 * torch.randn(D, generator=g)).to(DEV)
    C = torch.randn(B, H, L, D, generator=g).to(DEV)
    vx = torch.randn(x.shape, generator=g, dtype=torch.float64).to(DEV)
    vw = torch.randn(D, generator=g, dtype=torch.float64).to(DEV)
    pos = torch.arange(L, device=DEV)[None]
    f = lambda t: (qk_forward64(x.double() + t * vx, w.double() + t * vw, pos, inv, 1e-6)[0]
                   * C.double()).sum()
    h = 1e-4                                     # truncation h^2, rounding 2^-53 / h: 1e-8 each
    quotient = (f(h) - f(-h)) / (2 * h)
    dx, _, dw, _ = lops.qk_norm_rope_backward(x, None, w, None, 1e-6, inv, C, None)
    got = (dx.double() * vx).sum() + (dw.double() * vw).sum()
    scale = (dx.double() * vx).abs().sum() + (dw.double() * vw).abs().sum()
    assert abs(got - quotient) <= 1e-5 * scale


def test_qk_norm_rope_side_without_heads(lops):
    inv = lops.rope_inv_freq(64, 10000.0, DEV)
    w = torch.ones(64, device=DEV)
    q = torch.randn(1, 3, 5, 64, device=DEV)
    none = q[:, :0]
    for a, b in ((q, none), (none, q)):
        a2, b2 = lops.qk_norm_rope(a, b, w, w, 1e-6, inv)
        da, db, dwa, dwb = lops.qk_norm_rope_backward(a, b, w, w, 1e-6, inv, a2, b2)
        assert a2.shape == a.shape and db.shape == b.shape
        assert (dwa.abs().max() > 0) == (a is q) and (dwb.abs().max() > 0) == (b is q)
    alone, _ = lops.qk_norm_rope(q, None, w, None, 1e-6, inv)
    assert torch.equal(lops.qk_norm_rope(none, q, w, w, 1e-6, inv)[1], alone)


def test_qk_norm_rope_no_rows(lops):
    inv = lops.rope_inv_freq(64, 10000.0, DEV)
    w = torch.ones(64, device=DEV)
    q = torch.empty(2, 4, 0, 64, device=DEV)
    q2, k2 = lops.qk_norm_rope(q, q, w, w, 1e-6, inv)
    assert q2.shape == q.shape and k2.shape == q.shape
    _, _, dwq, dwk = lops.qk_norm_rope_backward(q, q, w, w, 1e-6, inv, q, q)
    assert not dwq.any() and not dwk.any()


# ---------------------------------------------------------------------------
# rows in 8 bits
# ---------------------------------------------------------------------------
def pack64(x, fmt):
    """(code values, scales) by the definition, in float64 on the CPU."""
    largest = torch.finfo(x.dtype).max
    x = x.cpu().double()
    d = x.shape[-1]
    xg = torch.nn.functional.pad(x, (0, -d % 128)).unflatten(-1, (-1, 128))
    top = xg.abs().amax(-1)
    bad = ~xg.isfinite().all(-1)
    top = torch.where(bad, 1.0, top)
    if fmt == "int8":
        s = (top / 127).float().double().clamp_min(2.0 ** -126)
        code = torch.round(xg / s[..., None])
    else:
        e = torch.full_like(top, -126)
        for k in range(-126, 128):               # the smallest e with top <= 448 2^e
            e = torch.where(top > 448 * 2.0 ** k, k + 1, e)
        s = torch.exp2(e)
        r = xg / s[..., None]
        k = torch.frexp(r).exponent.double() - 1
        step = torch.exp2(k.clamp_min(-6) - 3)
        code = torch.round(r / step) * step
        code = torch.where(code.abs() * s[..., None] > largest, 240.0 * code.sign(), code)
    s = torch.where(bad, float("nan"), s)
    code = torch.where(bad[..., None], 0.0, code)
    return code.flatten(-2)[..., :d], s


def code_values(p):
    if p.format == "int8":
        return p.codes.view(torch.int8).cpu().double()
    return p.codes.view(torch.float8_e4m3fn).cpu().double()


def special_rows(dtype, dim):
    """Rows that a rounding can get wrong: zeros, one element, the type's
    extremes, values on and next to the border between two codes."""
    g = torch.Generator().manual_seed(dim)
    big = torch.finfo(dtype).max
    rows = [torch.zeros(dim), torch.randn(dim, generator=g), 1e-30 * torch.randn(dim, generator=g),
            torch.randn(dim, generator=g) * torch.logspace(-8, 4, dim),
            torch.full((dim,), big), -big * torch.rand(dim, generator=g),
            torch.full((dim,), torch.finfo(dtype).smallest_normal),
            torch.full((dim,), TINY[dtype])]
    border = torch.arange(dim) % 127 + 0.5       # ties at scale 1
    border[::128] = 127.0
    rows.append(border)
    up = torch.nextafter(border, torch.tensor(float("inf")))
    up[::128] = 127.0
    rows.append(up)
    down = torch.nextafter(border, torch.tensor(0.0))
    down[::128] = -127.0
    rows.append(-down)
    for top in (3.1, 0.77, 113.0):               # ties at scales that are not powers of two
        s = (torch.tensor(top, dtype=torch.float64) / 127).float()
        r = (torch.arange(dim) % 127 + 0.5) * s
        r[::128] = top
        rows.append(r)
    e4 = torch.tensor([448.0, 17.0, 19.0, 2.0 ** -10, 3 * 2.0 ** -10, 2.0 ** -9, 1.0625, 1.1875])
    rows.append(e4.repeat(-(-dim // 8))[:dim])
    rows.append(torch.tensor([450.0, 0.3, -5.0]).repeat(dim)[:dim])
    return torch.stack(rows).to(DEV, dtype)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [8, 120, 128, 136, 1000, 4096])
def test_quantize_rows_codes_are_exact(lops, dtype, fmt, dim):
    x = special_rows(dtype, dim)
    p = lops.quantize_rows(x, fmt)
    codes, scales = pack64(x, fmt)
    assert torch.equal(p.scales.cpu().double(), scales)
    assert torch.equal(code_values(p), codes)
    back = lops.dequantize_rows(p)
    value = codes.float() * scales.float().repeat_interleave(128, -1)[:, :dim]
    assert torch.equal(back.cpu(), value.to(dtype))
    assert torch.equal(lops.dequantize_rows(p, torch.float32).cpu(), value)
    assert p.nbytes() == x.numel() + 4 * x.shape[0] * -(-dim // 128)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_rows_random_rows_are_exact(lops, dtype, fmt):
    g = torch.Generator().manual_seed(11)
    x = torch.randn(700, 520, generator=g) * torch.exp(3 * torch.randn(700, 1, generator=g))
    x = x.clamp(-6e4, 6e4).to(DEV, dtype)
    p = lops.quantize_rows(x, fmt)
    codes, scales = pack64(x, fmt)
    assert torch.equal(p.scales.cpu().double(), scales) and torch.equal(code_values(p), codes)
    # half a step: 1 / 254 of the group's largest (int8), 2^-4 of the value (e4m3) or half a
    # step of e4m3's subnormals, 2^-10 of a scale that is at most max / 224; and the rounding
    # of code * s to dtype
    err = (lops.dequantize_rows(p, torch.float32).cpu().double() - x.cpu().double()).abs()
    top = torch.nn.functional.pad(x.cpu().double().abs(), (0, -520 % 128)).unflatten(
        -1, (-1, 128)).amax(-1).repeat_interleave(128, -1)[:, :520]
    bound = top / 254 if fmt == "int8" else torch.maximum(
        x.cpu().double().abs() * 2.0 ** -4, top / 224 * 2.0 ** -10)
    assert (err <= bound * (1 + 4 * U) + 2 * U * top).all()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_rows_non_finite_groups(lops, dtype, fmt):
    x = torch.randn(3, 384, device=DEV).to(dtype)
    x[0, 130] = float("nan")
    x[1, 5] = float("inf")
    x[2, 383] = float("-inf")
    back = lops.dequantize_rows(lops.quantize_rows(x, fmt))
    bad = torch.zeros(3, 3, dtype=torch.bool, device=DEV)
    bad[0, 1] = bad[1, 0] = bad[2, 2] = True
    groups = back.view(3, 3, 128)
    assert groups[bad].isnan().all() and groups[~bad].isfinite().all()


def norm64(h, w, eps):
    h = h.double()
    rstd = (h.square().mean(-1) + eps).rsqrt()
    return h * rstd[..., None] * w.double(), rstd


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lead,dim,with_res", [
    ((1,), 8, True), ((5,), 264, False), ((2, 19), 1032, True), ((131,), 4096, True),
    ((3,), 2048, False), ((7,), 96, True), ((0,), 64, True), ((3,), 8192, True)])
def test_rmsnorm_packed(lops, dtype, fmt, lead, dim, with_res):
    if dim == 8192 and dtype == torch.float32:
        pytest.skip("above one row's limit in float32")
    g = torch.Generator().manual_seed(dim)
    x, r = (torch.randn(lead + (dim,), generator=g).to(DEV, dtype) for _ in range(2))
    r = r if with_res else None
    w = (1 + 0.1 * torch.randn(dim, generator=g)).to(DEV, dtype)
    h, y, rstd, p = lops.rmsnorm_forward_packed(x, w, 1e-6, residual=r, format=fmt)
    assert torch.equal(h, (x.float() + r.float()).to(dtype) if with_res else x)
    alone = lops.quantize_rows(h, fmt)
    assert torch.equal(p.codes, alone.codes) and torch.equal(p.scales, alone.scales)
    # rstd: sums of dim / 32 squares a lane (at least one vector of 8) and 5 steps between
    # lanes, halved by the root; the mean, eps and rsqrtf 5 u; y two products more
    su = ((max(dim / 32, 8) + 6) / 2 + 5) * U
    want, wr = norm64(h, w, 1e-6)
    check(rstd, wr, torch.float32, su * wr, "rstd")
    check(y, want, dtype, (su + 2 * U) * want.abs(), "y")
    h2, y2, rstd2 = lops.rmsnorm_from_packed(p, w, 1e-6)
    assert torch.equal(h2, lops.dequantize_rows(p))
    want, wr = norm64(h2, w, 1e-6)
    check(rstd2, wr, torch.float32, su * wr, "rstd of the restored rows")
    check(y2, want, dtype, (su + 2 * U) * want.abs(), "y of the restored rows")


def silu64(g):
    return g / (1 + torch.exp(-g))


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lead,ffn", [((1,), 8), ((33,), 64), ((2, 30), 1000), ((57,), 11008),
                                      ((0,), 16), ((3,), 264)])
def test_swiglu_packed(lops, dtype, fmt, lead, ffn):
    g = torch.Generator().manual_seed(ffn)
    gu = (3 * torch.randn(lead + (2 * ffn,), generator=g)).to(DEV, dtype)
    dout = torch.randn(lead + (ffn,), generator=g).to(DEV, dtype)
    out, p = lops.swiglu_forward_packed(gu, fmt)
    assert p.shape == lead + (2, ffn)
    alone = lops.quantize_rows(gu.view(lead + (2, ffn)), fmt)
    assert torch.equal(p.codes, alone.codes) and torch.equal(p.scales, alone.scales)
    gate, up = gu.double().chunk(2, -1)
    want = silu64(gate) * up
    # expf 2 u and its argument's rounding, 1 + e, the quotient, two products: below 16 u
    check(out, want, dtype, 16 * U * want.abs(), "out")
    dgu, again = lops.swiglu_backward_packed(p, dout)
    value = lops.dequantize_rows(p, torch.float32).double()
    gate, up, d = value[..., 0, :], value[..., 1, :], dout.double()
    s = 1 / (1 + torch.exp(-gate))
    check(again, silu64(gate) * up, dtype, 16 * U * (silu64(gate) * up).abs(), "out again")
    dg = d * up * s * (1 + gate * (1 - s))
    dgmag = (d * up * s).abs() * (1 + gate.abs())     # 1 - s cancels: its error is 8 u of 1
    check(dgu[..., :ffn], dg, dtype, 32 * U * dgmag, "dgate")
    du = d * gate * s
    check(dgu[..., ffn:], du, dtype, 16 * U * du.abs(), "dup")
    dgu2, none = lops.swiglu_backward_packed(p, dout, recompute=False)
    assert none is None and torch.equal(dgu2, dgu)


def test_swiglu_packed_large_gates(lops):
    """exp overflows for gates below -88: silu and its derivative go to zero."""
    gu = torch.tensor([[-200.0, -100.0, -89.0, -88.0, 88.0, 100.0, 200.0, 0.0] + [2.0] * 8],
                      device=DEV)
    out, p = lops.swiglu_forward_packed(gu, "e4m3")
    dgu, _ = lops.swiglu_backward_packed(p, torch.ones(1, 8, device=DEV))
    assert out.isfinite().all() and dgu.isfinite().all()
    assert out[0, 0].abs() < 1e-30 and dgu[0, 0].abs() < 1e-30


def test_swiglu_packed_gradient_is_the_difference_quotient(lops):
    g = torch.Generator().manual_seed(9)
    gu = torch.randn(5, 2 * 40, generator=g).to(DEV)
    C = torch.randn(5, 40, generator=g).to(DEV)
    _, p = lops.swiglu_forward_packed(gu, "int8")
    dgu, _ = lops.swiglu_backward_packed(p, C)
    at = lops.dequantize_rows(p, torch.float32).double()
    v = torch.randn(5, 80, generator=g, dtype=torch.float64).to(DEV)

    def f(t):
        z = at.flatten(-2) + t * v
        return (silu64(z[:, :40]) * z[:, 40:] * C.double()).sum()

    h = 1e-4
    got = (dgu.double() * v).sum()
    assert abs(got - (f(h) - f(-h)) / (2 * h)) <= 1e-5 * (dgu.double() * v).abs().sum()


# ---------------------------------------------------------------------------
# streams, capture, refusals
# ---------------------------------------------------------------------------
def all_ops(lops, seed):
    """One call of every operator; returns its outputs."""
    g = torch.Generator().manual_seed(seed)
    dt = torch.bfloat16
    ids = torch.randint(0, 300, (2, 900), generator=g).to(DEV)
    w = torch.randn(300, 256, generator=g).to(DEV, dt)
    nw = torch.randn(256, generator=g).to(DEV, dt)
    hw = torch.randn(64, generator=g).to(DEV, dt)
    inv = lops.rope_inv_freq(64, 10000.0, DEV)

    def run():
        e = lops.embedding_forward(ids, w, 2.0)
        h, y, rstd, p = lops.rmsnorm_forward_packed(e, nw, 1e-6, residual=e, format="int8")
        q = y.view(2, 900, 4, 64).transpose(1, 2)
        q2, k2 = lops.qk_norm_rope(q, q, hw, hw, 1e-6, inv)
        dq, dk, dwq, dwk = lops.qk_norm_rope_backward(q, q, hw, hw, 1e-6, inv, q2, k2)
        out, pm = lops.swiglu_forward_packed(y, "e4m3")
        dgu, _ = lops.swiglu_backward_packed(pm, out)
        h2, y2, _ = lops.rmsnorm_from_packed(p, nw, 1e-6)
        dw = lops.embedding_backward(ids, dgu, 300, 2.0)
        # more tokens than one launch takes: the general sort
        dws = [lops.embedding_backward(ids.repeat(1, n), dgu.repeat(1, n, 1), 300, 2.0)
               for n in (2, 3)]
        return [e, h, y, q2, k2, dq, dk, dwq, dwk, out, dgu, h2, y2, dw] + dws

    return run, (ids, w)


def test_operators_on_another_stream_and_captured(lops):
    """The same results on a side stream, and from two replays of two graphs
    captured one after the other (their workspaces are their own)."""
    runs = [all_ops(lops, s) for s in (1, 2)]
    want = [r() for r, _ in runs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [r() for r, _ in runs]
    side.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    graphs, outs = [], []
    for r, _ in runs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(r())
        graphs.append(graph)
    for _ in range(2):
        for graph in graphs:
            graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(want, outs):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    # new tokens in the captured buffer
    ids, w = runs[0][1]
    ids.copy_(ids.flip(1))
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0][0], lops.embedding_forward(ids, w, 2.0))


@pytest.mark.parametrize("n", [2560, 2561])       # sorted by one CTA, by several
def test_sorted_embedding_gradient_captured(lops, n):
    """Replays follow the ids and gradients that the inputs hold by then."""
    g = torch.Generator().manual_seed(n)
    cases = [(torch.randint(0, 5000, (n,), generator=g).to(DEV),
              torch.randn(n, 264, generator=g).to(DEV)) for _ in range(3)]
    want = [lops.embedding_backward(i, d, 5000, 0.5) for i, d in cases]
    ids, dy = (t.clone() for t in cases[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dw = lops.embedding_backward(ids, dy, 5000, 0.5)
    for (i, d), w in list(zip(cases, want)) * 2:
        ids.copy_(i)
        dy.copy_(d)
        graph.replay()
        assert torch.equal(dw, w)


def test_offsets_beyond_32_bits(lops):
    """Tensors of more than 2^32 bytes and 2^31 elements: the last rows come
    out as from a small tensor that holds them alone."""
    dt = torch.bfloat16
    rows, d = 540_000, 4096
    big = torch.empty(rows, d, device=DEV, dtype=dt)
    big[-40:] = torch.randn(40, d, device=DEV).to(dt)
    tail = big[-40:].clone()
    ids = torch.tensor([rows - 1, rows - 40, 0, rows - 7], device=DEV)
    out = lops.embedding_forward(ids, big, 1.0)
    assert torch.equal(out[[0, 1, 3]], tail[[39, 0, 33]])
    for n in (1, 3000):       # one launch, and sorted tokens
        dw = lops.embedding_backward(ids.repeat(n), tail[:4].repeat(n, 1), rows)
        small = lops.embedding_backward((ids - (rows - 40)).clamp_min(0)[[0, 1, 3]].repeat(n),
                                        tail[[0, 1, 3]].repeat(n, 1), 40)
        assert torch.equal(dw[-40:], small) and not dw[-60:-40].any() and dw[0].any()
        del dw
    for fmt in ("int8", "e4m3"):
        p, q = lops.quantize_rows(big, fmt), lops.quantize_rows(tail, fmt)
        assert torch.equal(p.codes[-40:], q.codes) and torch.equal(p.scales[-40:], q.scales)
        assert torch.equal(lops.dequantize_rows(p)[-40:], lops.dequantize_rows(q))
        del p
    w = torch.ones(d, device=DEV, dtype=dt)
    got = lops.rmsnorm_forward_packed(big, w, 1e-6)
    want = lops.rmsnorm_forward_packed(tail, w, 1e-6)
    assert torch.equal(got[1][-40:], want[1]) and torch.equal(got[3].codes[-40:], want[3].codes)
    back = lops.rmsnorm_from_packed(got[3], w, 1e-6)[1][-40:]
    assert torch.equal(back, lops.rmsnorm_from_packed(want[3], w, 1e-6)[1])
    del got
    out, p = lops.swiglu_forward_packed(big)
    out2, p2 = lops.swiglu_forward_packed(tail)
    assert torch.equal(out[-40:], out2)
    dgu, _ = lops.swiglu_backward_packed(p, out)
    assert torch.equal(dgu[-40:], lops.swiglu_backward_packed(p2, out2)[0])
    del dgu, out, p
    hw = torch.ones(128, device=DEV, dtype=dt)
    inv = lops.rope_inv_freq(128, 10000.0, DEV)
    q = big.view(rows, 32, 128).transpose(0, 1)[None]
    pos = torch.arange(rows, device=DEV)
    q2, _ = lops.qk_norm_rope(q, None, hw, None, 1e-6, inv, positions=pos)
    want, _ = lops.qk_norm_rope(q[:, :, -40:], None, hw, None, 1e-6, inv, positions=pos[-40:])
    assert torch.equal(q2[:, :, -40:], want)
    dq, _, _, _ = lops.qk_norm_rope_backward(q, None, hw, None, 1e-6, inv, q2, None, positions=pos)
    want, _, _, _ = lops.qk_norm_rope_backward(q[:, :, -40:], None, hw, None, 1e-6, inv, want, None,
                                               positions=pos[-40:])
    assert torch.equal(dq[:, :, -40:], want)


def test_refusals(lops, esa_mod):
    x = torch.randn(4, 64, device=DEV)
    w = torch.ones(64, device=DEV)
    ids = torch.zeros(4, dtype=torch.int64, device=DEV)
    err = esa_mod._lib.EsaError
    with pytest.raises(TypeError):
        lops.embedding_forward(ids.float(), x)
    with pytest.raises(RuntimeError):
        lops.embedding_forward(ids.cpu(), x)
    with pytest.raises(err):
        lops.embedding_forward(ids, torch.randn(4, 6, device=DEV))      # 24-byte rows
    with pytest.raises(ValueError):
        lops.embedding_forward(ids, torch.randn(4, 128, device=DEV)[:, :64])
    with pytest.raises(err):
        lops.embedding_forward(ids, x, float("nan"))
    with pytest.raises(ValueError):
        lops.embedding_backward(ids, x[:3], 10)
    with pytest.raises(ValueError):
        lops.embedding_backward(ids, x, 10, padding_idx=10)
    with pytest.raises(TypeError):
        lops.embedding_backward(ids, x.double(), 10)
    q = torch.randn(1, 2, 3, 64, device=DEV)
    inv = lops.rope_inv_freq(64, 10000.0, DEV)
    bad = dict(k=q[:, :, :2])
    with pytest.raises(ValueError):
        lops.qk_norm_rope(q, bad["k"], w, w, 1e-6, inv)
    with pytest.raises(ValueError):
        lops.qk_norm_rope(q, q, w, None, 1e-6, inv)
    with pytest.raises(ValueError):
        lops.qk_norm_rope(q, None, w.bfloat16(), None, 1e-6, inv)
    with pytest.raises(ValueError):
        lops.qk_norm_rope(q, None, w, None, 1e-6, inv[:5])
    with pytest.raises(ValueError):
        lops.qk_norm_rope(q, None, w, None, 1e-6, inv, positions=torch.arange(4, device=DEV))
    with pytest.raises(ValueError):
        lops.qk_norm_rope(q, None, w, None, 1e-6, inv, q_out=q[:, :1])
    with pytest.raises(ValueError):
        lops.qk_norm_rope(q.transpose(2, 3).contiguous().transpose(2, 3), None, w, None, 1e-6, inv)
    with pytest.raises(err):
        lops.qk_norm_rope(q, None, w, None, -1.0, inv)
    with pytest.raises(ValueError):
        lops.qk_norm_rope_backward(q, None, w, None, 1e-6, inv, q, q)
    with pytest.raises(ValueError):
        lops.quantize_rows(x, "int4")
    with pytest.raises(ValueError):
        lops.quantize_rows(x.t())
    with pytest.raises(TypeError):
        lops.quantize_rows(x.double())
    p = lops.quantize_rows(x)
    with pytest.raises(ValueError):
        lops.rmsnorm_from_packed(p, w[:32], 1e-6)
    with pytest.raises(ValueError):
        lops.swiglu_backward_packed(p, x)
    with pytest.raises(ValueError):
        lops.rmsnorm_forward_packed(x, w, 1e-6, residual=x[:2])
    with pytest.raises(ValueError):
        lops.dequantize_rows(lops.PackedRows(p.codes, p.scales[:2], "int8", torch.float32))
    assert esa_mod.ops.device_errors() == 0
