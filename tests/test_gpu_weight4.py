"""GPU: weights in 4 bits and products with them, against plain formulas in float64.

The codes are whole numbers and exact; a value is a code of 4 bits times a bfloat16
of 8 and exact in float32.  A product sums K exact terms in float32: at most one
unit in the last place (2 u, u = 2^-24) of a partial sum for each of the K / 16
steps of the matrix instruction (which may cut instead of rounding), the K / group
scaled sums and some 80 joins of partial sums, each at most the sum of the
magnitudes.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def lops():
    import elastic_sparse_attention_b200 as esa
    return esa.layer_ops


def decoded(w, group):
    """float64 values of the format's definition."""
    out = torch.empty(w.shape, dtype=torch.float64, device=w.device)
    for lo in range(0, w.shape[-1], group):
        x = w[..., lo:lo + group].double()
        top = x.abs().amax(-1, keepdim=True)
        s = (top.float() / torch.full_like(top, 7.0).float()).bfloat16().double().clamp_min(2.0 ** -126)
        v = torch.round(x / s) * s
        out[..., lo:lo + group] = torch.where((x.isfinite()).all(-1, keepdim=True), v, math.nan)
    return out


def weight(n, k, dtype, g, kind="normal"):
    w = 0.02 * torch.randn(n, k, generator=g)
    if kind == "ties":            # quotients that are half-integers, in every group
        w = torch.randint(-14, 15, (n, k), generator=g) / 2.0
        w[:, ::32] = 7.0
        w = w * 2.0 ** torch.randint(-5, 6, (n, 1), generator=g).float()
    elif kind == "ranges":        # zero groups, tiny and large ones
        e = torch.randint(-40, 14, (n, -(-k // 32)), generator=g).float()
        w = w * (2.0 ** e).repeat_interleave(32, -1)[:, :k]
        w[0] = 0
        w[-1, : k // 2] = 0
    return w.to(DEV, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("kind", ["normal", "ties", "ranges"])
@pytest.mark.parametrize("n,k", [(1, 8), (5, 40), (16, 128), (17, 136), (33, 1000), (130, 264),
                                 (1000, 2048)])
def test_codes_are_exact(lops, dtype, group, kind, n, k):
    g = torch.Generator().manual_seed(n * k + group)
    w = weight(n, k, dtype, g, kind)
    p = lops.quantize_weight4(w, group)
    assert p.shape == (n, k) and p.dtype == dtype
    want = decoded(w, group)
    assert torch.equal(lops.dequantize_weight4(p, torch.float32).double(), want)
    for out in DTYPES:
        assert torch.equal(lops.dequantize_weight4(p, out), want.float().to(out))


@pytest.mark.parametrize("dtype", DTYPES)
def test_extreme_groups(lops, dtype):
    w = torch.randn(20, 256, generator=torch.Generator().manual_seed(1)).to(DEV, dtype)
    w[1, 3] = math.nan
    w[2, 200] = math.inf
    w[3, 40] = -math.inf
    w[4] = torch.finfo(dtype).max
    w[5] = -torch.finfo(dtype).max
    w[6, :128] = torch.finfo(dtype).tiny
    w[7, 128:] = torch.finfo(dtype).smallest_normal * 3
    for group in (32, 64, 128):
        v = lops.dequantize_weight4(lops.quantize_weight4(w, group), torch.float32).double()
        want = decoded(w, group)
        assert torch.equal(v.isnan(), want.isnan())
        ok = ~want.isnan()
        assert torch.equal(v[ok], want[ok])
        assert torch.isfinite(v[4:]).all()
        x = torch.ones(2, 256, device=DEV).to(dtype)
        y = lops.linear4(x, lops.quantize_weight4(w[:4], group))
        assert y.isnan().tolist() == [[False, True, True, True]] * 2


def product_bound(x, v, group, dtype):
    terms = x.double().abs() @ v.abs().t()
    K = x.shape[-1]
    return 2 * U * (K / 16 + K / group + 80) * terms


def check(y, x, v, group, what):
    want = x.double() @ v.t()
    slack = product_bound(x, v, group, x.dtype)
    half_step = torch.finfo(x.dtype).eps / 2
    bound = half_step * (want.abs() + slack) + slack + 2.0 ** -24 * (x.dtype == torch.float16)
    assert y.dtype == x.dtype and y.shape == want.shape
    bad = ~((y.double() - want).abs() <= bound)
    assert not bad.any(), (what, int(bad.sum()), float((y.double() - want).abs().max()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,k", [(1, 8), (18, 40), (16, 128), (50, 264), (300, 1000), (129, 2056),
                                 (2600, 512), (40, 9000)])
def test_linear(lops, dtype, group, n, k):
    g = torch.Generator().manual_seed(n + k + group)
    w = weight(n, k, dtype, g)
    p = lops.quantize_weight4(w, group)
    v = decoded(w, group)
    for m in (1, 2, 3, 5, 6, 8, 9, 16, 17, 21, 22, 32, 33, 43, 64, 65, 130):
        if m > 9 and k == 9000 and group != 64:
            continue
        x = torch.randn(m, k, generator=g).to(DEV, dtype)
        y = lops.linear4(x, p)
        check(y, x, v, group, (m, n, k))
        assert torch.equal(y, lops.linear4(x, p))                # the same in every run
    assert lops.linear4(x[:0], p).shape == (0, n)
    assert torch.equal(lops.linear4(x[:6].view(2, 3, k), p).view(6, n), lops.linear4(x[:6], p))


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_large(lops, dtype):
    """The stack's shapes, and one that splits K over a whole cluster."""
    g = torch.Generator().manual_seed(0)
    for n, k, m in ((12288, 4096, 1), (4096, 11008, 32), (4096, 4096, 64), (24, 16384, 40)):
        w = weight(n, k, dtype, g)
        x = torch.randn(m, k, generator=g).to(DEV, dtype)
        check(lops.linear4(x, lops.quantize_weight4(w, 128)), x, decoded(w, 128), 128, (n, k, m))


def test_float32_rows_keep_their_bits(lops):
    """x with 24 significant bits and a wide range, against a weight of one code per
    row: the three 8-bit parts of x lose nothing.  What is left are the two float32
    additions that put 7 times them together: two halves of a unit."""
    k = 256
    w = torch.zeros(16, k, device=DEV)
    w[torch.arange(16), torch.arange(16) * 16] = 7.0
    p = lops.quantize_weight4(w, 128)
    g = torch.Generator().manual_seed(19)
    for m in (2, 3, 40):
        x = (torch.randn(m, k, generator=g) * 2.0 ** torch.randint(-60, 60, (m, k), generator=g).float())
        x = x.to(DEV)
        want = 7.0 * x[:, ::16].double()
        assert ((lops.linear4(x, p).double() - want).abs() <= 2 * U * (1 + 2.0 ** -7) * want.abs()).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [3, 30])
def test_infinite_and_nan_inputs(lops, dtype, m):
    w = torch.full((20, 200), 0.5, device=DEV).to(dtype)
    w[10:] = -0.5
    p = lops.quantize_weight4(w, 64)
    x = torch.randn(m, 200, device=DEV).to(dtype)
    x[1, 7] = math.inf
    x[2, 150] = math.nan
    y = lops.linear4(x, p)
    assert torch.isfinite(y[0]).all() and y[2].isnan().all()
    assert (y[1, :10] == math.inf).all() and (y[1, 10:] == -math.inf).all()


def test_refusals(lops):
    w = torch.randn(20, 64, device=DEV)
    p = lops.quantize_weight4(w)
    with pytest.raises(ValueError, match="group"):
        lops.quantize_weight4(w, 16)
    with pytest.raises(ValueError):
        lops.quantize_weight4(w[0])
    with pytest.raises(ValueError):
        lops.quantize_weight4(w[:0])
    with pytest.raises(ValueError):
        lops.quantize_weight4(w.t())
    with pytest.raises(TypeError):
        lops.quantize_weight4(w.double())
    with pytest.raises(ValueError):
        lops.linear4(torch.randn(2, 60, device=DEV), p)
    with pytest.raises(ValueError):
        lops.linear4(torch.randn(64, 2, device=DEV).t(), p)
    with pytest.raises(TypeError):
        lops.linear4(torch.randn(2, 64, device=DEV).double(), p)
    broken = lops.PackedWeight4(p.codes, p.scales, (40, 64), p.group, p.dtype)
    for call in (lambda: lops.linear4(torch.randn(2, 64, device=DEV), broken),
                 lambda: lops.dequantize_weight4(broken)):
        with pytest.raises(ValueError, match="fit"):
            call()
    with pytest.raises(RuntimeError):
        lops.linear4(torch.randn(2, 64), p)


def test_captured_beside_other_kernels(lops):
    """A chain of products whose kernels begin before the one before has ended, on
    inputs that change between replays."""
    g = torch.Generator().manual_seed(5)
    ps = [lops.quantize_weight4(weight(512, 512, torch.bfloat16, g), 64) for _ in range(6)]
    x = torch.randn(3, 512, generator=g).to(DEV, torch.bfloat16)

    def chain():
        y = x
        for p in ps:
            y = lops.linear4(y, p)
        return y
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        chain()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = chain()
    for seed in range(3):
        x.copy_(torch.randn(3, 512, generator=torch.Generator().manual_seed(seed)) * 10)
        graph.replay()
        want = x
        for p in ps:                    # one at a time
            want = lops.linear4(want, p)
            torch.cuda.synchronize()
        assert torch.equal(y, want)
    # weights made in the same stream right before their use
    for seed in range(3):
        w = weight(3000, 1024, torch.bfloat16, g)
        xx = torch.randn(2, 1024, generator=g).to(DEV, torch.bfloat16)
        y1 = lops.linear4(xx, lops.quantize_weight4(w, 128))
        check(y1, xx, decoded(w, 128), 128, "fresh")


@pytest.mark.parametrize("rows", [1, 24])
@pytest.mark.parametrize("how", ["quantize", "copy"])
def test_codes_made_by_the_kernel_before(lops, rows, how):
    """The product reads what the kernel right before it wrote: codes and scales of
    other weights put into the same memory, nothing waited for in between."""
    from elastic_sparse_attention_b200 import _lib
    g = torch.Generator(device=DEV).manual_seed(11)
    n, k = 4096, 1024
    x = torch.randn(rows, k, device=DEV, generator=g).bfloat16()
    weights = [torch.randn(n, k, device=DEV, generator=g).bfloat16() for _ in range(2)]
    packed = [lops.quantize_weight4(w) for w in weights]
    torch.cuda.synchronize()
    want = [lops.linear4(x, p) for p in packed]
    torch.cuda.synchronize()
    shared = lops.quantize_weight4(weights[0])
    lib = _lib.load()
    got = []
    for i in range(24):
        if how == "copy":
            shared.scales.copy_(packed[i % 2].scales)
            shared.codes.copy_(packed[i % 2].codes)
        else:
            _lib.launch(lib.esa_quantize_weight4, x.device, _lib.DTYPES[x.dtype], n, k,
                        shared.group, weights[i % 2].data_ptr(), shared.codes.data_ptr(),
                        shared.scales.data_ptr())
        got.append(lops.linear4(x, shared))
    for i, y in enumerate(got):
        assert torch.equal(y, want[i % 2]), i


def test_the_most_weight_rows(lops):
    """2^20 rows, 65536 tiles of 16: the last ones as if they were alone."""
    g = torch.Generator(device=DEV).manual_seed(12)
    w = torch.randn(1 << 20, 32, device=DEV, generator=g).bfloat16()
    x = torch.randn(2, 32, device=DEV, generator=g).bfloat16()
    p, last = lops.quantize_weight4(w, 32), lops.quantize_weight4(w[-32:].contiguous(), 32)
    assert torch.equal(p.codes[-2048:], last.codes)
    assert torch.equal(p.scales[-2:, :1], last.scales[:, :1])
    assert torch.equal(lops.dequantize_weight4(p)[-32:], lops.dequantize_weight4(last))
    assert torch.equal(lops.linear4(x, p)[:, -32:], lops.linear4(x, last))
