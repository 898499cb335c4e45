"""GPU: weights in 4 bits and products with them at the ends of their types' range."""
import math

import pytest
import torch

from test_gpu_weight4 import DEV, decoded

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lops():
    import elastic_sparse_attention_b200 as esa
    return esa.layer_ops


@pytest.mark.parametrize("rows", [1, 3, 30])
@pytest.mark.parametrize("bits", [0x7f800001, 0x7fc00000, 0x7fffffff, -0x007fffff, -0x00400000,
                                  0x7f80ffff, 0x7f810000])
def test_every_nan_of_float32_rows(lops, rows, bits):
    """Also one whose set bits are all among the low 16 of its 23."""
    w = torch.full((20, 200), 0.5, device=DEV)
    p = lops.quantize_weight4(w, 64)
    x = torch.randn(rows, 200, generator=torch.Generator().manual_seed(rows)).to(DEV)
    x.view(torch.int32)[0, 150] = bits
    assert x[0, 150].isnan()
    y = lops.linear4(x, p)
    assert y[0].isnan().all() and torch.isfinite(y[1:]).all()


@pytest.mark.parametrize("group", [32, 64, 128])
def test_the_largest_weights(lops, group):
    """7 steps of a group whose largest magnitude is bfloat16's largest value are
    1022 * 2^118, halfway between that value and 2^128: its rounding is infinity.  So
    in bfloat16 alone: no other value, and not in float32, where a product takes it as
    it is."""
    big = torch.finfo(torch.bfloat16).max
    w = torch.zeros(4, 128, device=DEV, dtype=torch.bfloat16)
    w[0, 3], w[1, 3] = big, -big
    w[2, 3] = torch.nextafter(torch.tensor(big, dtype=torch.bfloat16), torch.tensor(0.0, dtype=torch.bfloat16))
    w[3, 3] = 1.0
    p = lops.quantize_weight4(w, group)
    v = lops.dequantize_weight4(p, torch.float32)
    assert torch.equal(v.double(), decoded(w, group)) and torch.isfinite(v).all()
    assert float(v[0, 3]) == 1022 * 2.0 ** 118
    h = lops.dequantize_weight4(p)
    assert h[0, 3] == math.inf and h[1, 3] == -math.inf and torch.isfinite(h[2:]).all()
    x = torch.zeros(1, 128, device=DEV, dtype=torch.bfloat16)
    x[0, 3] = 0.25
    assert lops.linear4(x, p)[0, :2].tolist() == [2.0 ** 126, -2.0 ** 126]
    for dtype in (torch.float16, torch.float32):      # the largest values there stay finite
        w = torch.full((1, 128), torch.finfo(dtype).max, device=DEV, dtype=dtype)
        assert torch.isfinite(lops.dequantize_weight4(lops.quantize_weight4(w, group))).all()


def test_captured_on_two_streams_that_join(lops):
    """Products and scores of two branches of one graph, then a product that needs both,
    with copies in between: kernels that may start early have several predecessors, not
    all of them kernels."""
    g = torch.Generator().manual_seed(21)
    ps = [lops.quantize_weight4((0.05 * torch.randn(512, 512, generator=g)).to(DEV, torch.bfloat16), 64)
          for _ in range(4)]
    xs = [torch.randn(m, 512, generator=g).to(DEV, torch.bfloat16) for m in (3, 20)]
    tokens = torch.randint(0, 512, (20,), generator=g).to(DEV)
    side = torch.cuda.Stream()

    def run(two):
        main = torch.cuda.current_stream()
        a = lops.linear4(xs[0], ps[0])
        if two:
            side.wait_stream(main)
        with torch.cuda.stream(side if two else main):
            b = lops.linear4(lops.linear4(xs[1], ps[1]), ps[2])
            scores = lops.token_logprobs(b, tokens, top_k=4)
        a = lops.linear4(a, ps[3])
        if two:
            main.wait_stream(side)
        both = torch.cat([a, b])
        y = lops.linear4(both, ps[0])
        both.copy_(y)
        return lops.linear4(both, ps[1]), scores.logprobs, scores.top_ids

    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        run(True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(True)
    for seed in range(4):
        for x in xs:
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        for t, want in zip(got, run(False)):
            assert torch.equal(t, want)
