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
