"""GPU: sums of the layer operators' gradients on inputs whose float32 sums are
exact, so that a row that is lost, counted twice or taken from an earlier call
shows in the result whatever the rounding.

dy holds small integers and the scale is a power of two: every partial sum is
an integer below 2^24, which float32 holds exactly in any order, and the one
rounding to dw's type is the rounding of the exact value.
"""
import pytest
import torch

DEV = "cuda:0"


def exact_gradient(ids, dy, V, scale, dtype):
    """dw of integer-valued dy, rounded once."""
    dw = torch.zeros(V, dy.shape[1], dtype=torch.float64, device=dy.device)
    return (dw.index_add_(0, ids, dy.double()) * scale).to(dtype)


@pytest.fixture(scope="module")
def lops():
    import elastic_sparse_attention_b200 as esa
    return esa.layer_ops


@pytest.mark.gpu
@pytest.mark.parametrize("n,V,d", [
    (2500, 40000, 8), (9000, 500, 264), (9000, 70000, 16), (9000, 300000, 8)])
def test_embedding_gradients_in_a_row(lops, n, V, d):
    """Calls issued back to back (one CTA's sort; one, two and three digits),
    whose sorted pairs lie where the call before had its own."""
    g = torch.Generator().manual_seed(n + V)
    calls = []
    for _ in range(12):
        ids = torch.randint(0, V, (n,), generator=g).to(DEV)
        dy = torch.randint(-3, 4, (n, d), generator=g).float().to(DEV)
        calls.append((ids, dy))
    want = [exact_gradient(i, t, V, 0.5, torch.float32) for i, t in calls]
    torch.cuda.synchronize()
    got = [lops.embedding_backward(i, t, V, 0.5) for i, t in calls]
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_qk_weight_gradients_in_a_row(lops):
    """The weight sums of calls issued back to back are those of the calls made
    one at a time."""
    g = torch.Generator().manual_seed(4)
    w = (1 + 0.1 * torch.randn(64, generator=g)).to(DEV)
    inv = lops.rope_inv_freq(64, 10000.0, DEV)
    q = torch.randn(1, 4, 700, 64, generator=g).to(DEV)
    douts = [torch.randn(1, 4, 700, 64, generator=g).to(DEV) for _ in range(12)]

    def call(do):
        return lops.qk_norm_rope_backward(q, q, w, w, 1e-6, inv, do, do)[2:]

    want = []
    for do in douts:
        want.append(call(do))
        torch.cuda.synchronize()
    got = [call(do) for do in douts]
    for (a, b), (c, d) in zip(got, want):
        assert torch.equal(a, c) and torch.equal(b, d)


def border_rows(dtype):
    """Rows of one group whose int8 scale is just above 2^-126 with an odd last
    bit, so that half of it is no float32, and values next to the border between
    two codes; and the codes by float64, whose quotients keep a distance of
    2^-25 from the border that float64 resolves."""
    g = torch.Generator().manual_seed(21)
    rows = 256
    m = (1 << 23) + 2 * torch.randint(0, 1 << 22, (rows, 1), generator=g) + 1   # s = m 2^-149
    k = torch.randint(0, 126, (rows, 128), generator=g)
    x = ((2 * k + 1) * m + torch.randint(0, 2, k.shape, generator=g) * 2 - 1).double() * 2.0 ** -150
    x = x * (torch.randint(0, 2, k.shape, generator=g) * 2 - 1)
    x[:, :1] = 127 * m.double() * 2.0 ** -149
    x = x.to(dtype)
    s = (x.double().abs().amax(-1, keepdim=True) / 127).float().double().clamp_min(2.0 ** -126)
    return x, torch.round(x.double() / s), s


def test_border_rows_reach_the_border():
    x, _, s = border_rows(torch.float32)
    steps = (x.double().abs() / s - 0.5).frac().sub(0.5).abs()
    odd = (s * 2.0 ** 149).long() & 1 == 1
    assert (odd & (s < 2.0 ** -125)).sum() > 100
    assert (0.5 - steps < 2.0 ** -23).sum() > 2000


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_int8_borders_at_the_smallest_scales(lops, dtype):
    x, codes, s = border_rows(dtype)
    p = lops.quantize_rows(x.to(DEV), "int8")
    assert torch.equal(p.scales.cpu().double(), s)
    assert torch.equal(p.codes.view(torch.int8).cpu().double(), codes)


# ---------------------------------------------------------------------------
# every row of the embedding gradient, at the borders of the pieces
# ---------------------------------------------------------------------------
def pieces_case(P, lengths, n_max, seed):
    """Token ids, shuffled, whose sorted list has a run of each length beginning at
    each offset within a piece of P entries; every second vocabulary entry is
    absent.  (ids, V)"""
    g = torch.Generator().manual_seed(seed)
    runs, at = [], 0
    for length in lengths:
        for offset in range(P):
            fill = (offset - at) % P
            while fill > 0:                       # short runs up to the offset
                step = min(fill, int(torch.randint(1, P, (), generator=g)))
                runs.append(step)
                fill -= step
                at += step
            runs.append(length)
            at += length
    assert at <= n_max, at
    tokens = 2 * torch.arange(len(runs)) + 1
    ids = tokens.repeat_interleave(torch.tensor(runs))
    return ids[torch.randperm(at, generator=g)], 2 * len(runs) + 2


def odd_rows(n, d, g):
    """Rows of +-1: no sum without one of them is the same."""
    return (2 * torch.randint(0, 2, (n, d), generator=g) - 1).float()


# Pieces of 16, 32 and 64 entries: by width and token count.  Each with runs of
# up to three pieces; and long runs, which several pieces share.
PIECES = {
    "narrow-16": (16, 64, 1 << 20, 2561), "wide-16": (16, 264, 8192, 2561),
    "wide-32": (32, 264, 65536, 8193), "wide-64": (64, 264, 1 << 20, 65537),
    "one-cta-16": (16, 264, 2560, 1025),
}


def pieces_ids(name):
    P, d, n_max, n_min = PIECES[name]
    lengths = [P - 1, P, P + 1, 2 * P - 1, 2 * P, 2 * P + 1, 3 * P, 3 * P + 1, 1]
    if name == "one-cta-16":
        lengths = [P - 1, P, P + 1, 2 * P + 1]
    ids, V = pieces_case(P, lengths, n_max, P + d)
    g = torch.Generator().manual_seed(d)
    more = max(n_min - ids.numel(), 0)            # one long run brings it to the length wanted
    room = n_max - ids.numel() - more
    more += min(room, 40 * P + 3)
    ids = torch.cat([ids, torch.full((more,), V - 2)])
    ids = ids[torch.randperm(ids.numel(), generator=g)]
    assert n_min <= ids.numel() <= n_max
    return ids, V, d


def lost_unseen(ids, dy, V, scale, dtype):
    """Rows of dy without which the rounded gradient would be the same: without a
    row it differs from the whole by that row, in its token's entry alone."""
    whole = exact_gradient(ids, dy, V, 1.0, torch.float64)[ids]
    without = ((whole - dy.double()) * scale).to(dtype)
    return (without == (whole * scale).to(dtype)).all(1).nonzero().flatten()


@pytest.mark.parametrize("name", PIECES)
def test_every_lost_row_would_show(name):
    """The oracle without any one of the rows differs from the whole."""
    ids, V, d = pieces_ids(name)
    dy = odd_rows(ids.numel(), 8, torch.Generator().manual_seed(1))
    for dtype in (torch.float32, torch.bfloat16):
        assert not lost_unseen(ids, dy, V, 0.25, dtype).numel()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("name", PIECES)
def test_embedding_gradient_at_piece_borders(lops, name, dtype):
    ids, V, d = pieces_ids(name)
    ids = ids.to(DEV)
    dy = odd_rows(ids.numel(), d, torch.Generator().manual_seed(2)).to(DEV)
    for pad in (None, 7):
        want = exact_gradient(ids, dy, V, 0.25, dtype)
        if pad is not None:
            want[pad] = 0
        got = lops.embedding_backward(ids, dy.to(dtype), V, 0.25, padding_idx=pad)
        assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,V,d", [
    (1, 40, 8), (31, 7, 64), (130, 3, 520), (1000, 33, 520), (1024, 900, 1032), (1024, 1, 264),
    (2047, 64, 64), (2048, 5, 256), (2048, 3000, 8),
    # the general sort with one digit, two and three, all tokens the same
    (70001, 1, 264), (9000, 2, 1032), (20000, 511, 16), (20000, 262143, 8), (66000, 300000, 264)])
def test_embedding_gradient_is_exact_on_integers(lops, dtype, n, V, d):
    g = torch.Generator().manual_seed(n + V + d)
    ids = torch.randint(0, V, (n,), generator=g).to(DEV)
    dy = odd_rows(n, d, g).to(DEV)
    assert torch.equal(lops.embedding_backward(ids, dy.to(dtype), V, 2.0),
                       exact_gradient(ids, dy, V, 2.0, dtype))


# ---------------------------------------------------------------------------
# every row of the query / key norm's weight gradients
# ---------------------------------------------------------------------------
U = 2.0 ** -24
WEIGHT_SHAPES = [(1, 1, 32, 8, 128), (2, 333, 4, 2, 64), (3, 5, 3, 1, 16), (2, 40, 6, 2, 128),
                 (1, 2100, 8, 2, 128), (3, 2400, 1, 1, 16), (2, 5003, 3, 1, 32),
                 (1, 9001, 2, 1, 128), (5, 1500, 5, 2, 64), (1, 4800, 5, 1, 32),
                 (2, 700, 16, 4, 128), (1, 900, 40, 8, 64)]


def weight_case(dtype, B, L, H, D, seed, only=None):
    """(x, dout), [B, H, L, D]; ``only``: the tokens b * L + l whose dout is not zero."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, L, H, D, generator=g).to(dtype)
    dout = torch.randn(B, L, H, D, generator=g).to(dtype)
    if only is not None:
        keep = torch.zeros(B * L, dtype=torch.bool)
        keep[only] = True
        dout[~keep.view(B, L)] = 0
    return x.transpose(1, 2), dout.transpose(1, 2)


def weight_gradient64(x, dout, inv, eps=1e-6):
    """(terms of dw [B, H, L, D], bound of each one's float32 error over U)."""
    xh = x.double() * (x.double().square().mean(-1, keepdim=True) + eps).rsqrt()
    ang = torch.arange(x.shape[2], device=x.device).double()[:, None] * inv.double()
    c, s = ang.cos(), ang.sin()
    a, b = dout.double().chunk(2, -1)
    gr = torch.cat([a * c + b * s, b * c - a * s], -1)
    mag = torch.cat([a.abs() + b.abs()] * 2, -1) * xh.abs()
    return gr * xh, mag


def summation_depth(B, L, Hq, Hk, D, side):
    """Additions that a term of dw passes through at most: a lane's own rows (one
    in every 32 / threads-per-row of a warp's, over the side's warps, of which a
    CTA has 4; whole rounds of up to 4), the lanes of a warp (5), its CTA's warps
    (4), a warp's share of the CTAs' sums and the 32 warps of that."""
    rows = B * L * (Hq if side == 0 else Hk)
    ctas = max(2, min(444, -(-B * L * (Hq + Hk) // 4)))
    share = ctas * (Hq if side == 0 else Hk) / (Hq + Hk)     # at least half of it: see below
    lanes = max(1, share / 2) * 4 * 32 / (D / 8)
    return rows / lanes + 32 + 5 + 4 + ctas / 32 + 1 + 32


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,L,Hq,Hk,D", WEIGHT_SHAPES)
def test_qk_weight_gradient_of_single_tokens(lops, dtype, B, L, Hq, Hk, D):
    """dout is zero but for a few tokens, at the ends of the sequences and in
    between: a sum that misses one of them is off by a large part of itself."""
    inv = lops.rope_inv_freq(D, 10000.0, DEV)
    w = torch.ones(D, device=DEV, dtype=dtype)
    n = B * L
    for seed in range(4):
        g = torch.Generator().manual_seed(100 + seed)
        picks = torch.cat([torch.tensor([0, n - 1, L - 1, n - L]),
                           torch.randint(0, n, (2,), generator=g)]).unique()
        if seed == 3:
            picks = torch.arange(max(0, n - 9), n)            # the last tasks
        (q, dq), (k, dk) = (tuple(t.to(DEV) for t in weight_case(dtype, B, L, H, D, seed + H, picks))
                            for H in (Hq, Hk))
        _, _, dwq, dwk = lops.qk_norm_rope_backward(q, k, w, w, 1e-6, inv, dq, dk)
        for side, (dw, x, do) in enumerate(((dwq, q, dq), (dwk, k, dk))):
            terms, mag = weight_gradient64(x, do, inv)
            want, mag = terms.sum((0, 1, 2)), mag.sum((0, 1, 2))
            # 64 u of each term (as for dx), the sums, the one rounding
            slack = (64 + summation_depth(B, L, Hq, Hk, D, side)) * U * mag
            bound = slack + torch.finfo(dtype).eps / 2 * (want.abs() + slack)
            assert ((dw.double() - want).abs() <= bound).all(), (seed, side)


@pytest.mark.gpu
@pytest.mark.parametrize("B,L,Hq,Hk,D", WEIGHT_SHAPES)
def test_qk_weight_gradient_misses_no_row(lops, B, L, Hq, Hk, D):
    """Full dout in float32: the bound by the depth of the sums is smaller than
    what the mean row adds, so that the sum without any one row exceeds it."""
    inv = lops.rope_inv_freq(D, 10000.0, DEV)
    w = torch.ones(D, device=DEV)
    (q, dq), (k, dk) = (tuple(t.to(DEV) for t in weight_case(torch.float32, B, L, H, D, 7 * H))
                        for H in (Hq, Hk))
    _, _, dwq, dwk = lops.qk_norm_rope_backward(q, k, w, w, 1e-6, inv, dq, dk)
    for side, (dw, x, do) in enumerate(((dwq, q, dq), (dwk, k, dk))):
        terms, mag = weight_gradient64(x, do, inv)
        want, mag = terms.sum((0, 1, 2)), mag.sum((0, 1, 2))
        slack = (64 + summation_depth(B, L, Hq, Hk, D, side)) * U * mag
        bound = slack + U * (want.abs() + slack)
        # what a lost row would leave, in the column where it is largest over its bound
        lost = (terms.abs() / (2 * bound)).amax(-1)
        assert (lost > 1).all(), float(lost.min())
        assert ((dw.double() - want).abs() <= bound).all(), side


def test_the_largest_scale_by_arithmetic():
    """127 * f32(a / 127) passes the largest float32 for that value alone: in units
    of 2^98 it is 2^30 - 64 and its neighbours are 64 apart; 127 s rounds to
    infinity from 2^30 - 32 on, which takes s >= 8454660, so a / 127 >= 8454659.5,
    so a >= 2^30 - 67.5."""
    big = torch.tensor(torch.finfo(torch.float32).max)
    below = torch.nextafter(big, torch.tensor(0.0))
    for a, finite in ((big, False), (below, True)):
        s = (a.double() / 127).float()
        assert (127 * s).isfinite().item() == finite
    assert 127 * 8454660 >= 2 ** 30 - 32 > 127 * 8454659


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_the_largest_values_come_back_finite(lops, fmt):
    """All but the largest float32 in int8, whose documented value is infinite."""
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        big = torch.tensor(torch.finfo(dtype).max, dtype=dtype)
        x = torch.randn(4, 128, generator=torch.Generator().manual_seed(1)).to(dtype)
        x[0, 5], x[1, 9] = big, -big
        x[2, 3] = x[2, 4] = torch.nextafter(big, torch.tensor(0, dtype=dtype))
        back = lops.dequantize_rows(lops.quantize_rows(x.to(DEV), fmt)).cpu()
        if fmt == "int8" and dtype == torch.float32:
            assert back[0, 5] == float("inf") and back[1, 9] == float("-inf")
            back[0, 5] = back[1, 9] = 0
        assert back.isfinite().all()


@pytest.mark.gpu
def test_calls_on_two_streams_and_threads(lops):
    """Calls in flight at the same time have their workspaces to themselves."""
    import threading
    g = torch.Generator().manual_seed(6)
    w = (1 + 0.1 * torch.randn(64, generator=g)).to(DEV)
    inv = lops.rope_inv_freq(64, 10000.0, DEV)
    jobs = []
    for n in (3000, 9000):
        ids = torch.randint(0, 5000, (n,), generator=g).to(DEV)
        dy = odd_rows(n, 264, g).to(DEV)
        q = torch.randn(1, 4, n, 64, generator=g).to(DEV)

        def job(ids=ids, dy=dy, q=q):
            return (lops.embedding_backward(ids, dy, 5000, 0.5),
                    *lops.qk_norm_rope_backward(q, q, w, w, 1e-6, inv, q, q))
        jobs.append(job)
    want = [j() for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    got = [[], []]

    def go(k):
        with torch.cuda.stream(streams[k]):
            for _ in range(20):
                got[k].append(jobs[k]())
        streams[k].synchronize()

    threads = [threading.Thread(target=go, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for k in range(2):
        assert len(got[k]) == 20
        for out in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(out, want[k]))
