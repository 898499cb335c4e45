"""GPU: log probabilities and their gradient at the upper end of the logits' types,
against plain formulas in float64; bounds as in test_gpu_score.py."""
import math

import pytest
import torch

from test_gpu_score import DEV, DTYPES, TINY, U, Exact, close

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def esa():
    import elastic_sparse_attention_b200 as mod
    return mod


def rows_of(kind, rows, V, dtype, g):
    """Each row has its largest logit in a place of its own."""
    x = 3 * torch.randn(rows, V, generator=g, dtype=torch.float64)
    top = torch.finfo(dtype).max
    at = torch.randint(0, V, (rows,), generator=g)
    if kind == "among -infinities":
        x[torch.rand(rows, V, generator=g) < 0.5] = -math.inf
    elif kind == "alone among -infinities":
        x[:] = -math.inf
    elif kind == "among lowest":
        x[torch.rand(rows, V, generator=g) < 0.7] = torch.finfo(dtype).min
    elif kind == "spread":
        x = (2 * torch.rand(rows, V, generator=g, dtype=torch.float64) - 1) * top
    elif kind == "three quarters":
        top = 0.75 * top
        x[torch.rand(rows, V, generator=g) < 0.5] = -math.inf
    elif kind == "all":
        x[:] = top
    elif kind == "far below":          # a whole row next to the type's lowest value
        x = torch.finfo(dtype).min * (1 - 0.5 * torch.rand(rows, V, generator=g, dtype=torch.float64))
        top = 0.5 * torch.finfo(dtype).min
    elif kind == "two":
        x[torch.arange(rows), torch.randint(0, V, (rows,), generator=g)] = top
    x[torch.arange(rows), at] = top
    return x.to(dtype).to(DEV), at.to(DEV)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["normal", "among -infinities", "alone among -infinities",
                                  "among lowest", "spread", "three quarters", "all", "far below",
                                  "two"])
@pytest.mark.parametrize("rows,V", [(2, 1), (3, 7), (5, 100), (40, 513), (2, 4097), (3, 32000),
                                    (160, 5000)])
def test_the_largest_logits(esa, dtype, kind, rows, V):
    g = torch.Generator().manual_seed(rows + V)
    x, at = rows_of(kind, rows, V, dtype, g)
    tokens = torch.randint(0, V, (rows,), generator=g).to(DEV)
    tokens[0] = at[0]
    top = min(V, 5)
    e = Exact(x, tokens)
    r = esa.layer_ops.token_logprobs(x, tokens, top_k=top)
    # what is below float32's range is its -infinity
    want = e.token_lp.float().double()
    close(r.logprobs, want, e.lp_bound(e.token_lp[:, None])[:, 0], "logprobs")
    close(r.entropy, e.entropy, e.err_entropy, "entropy")
    assert torch.isfinite(r.entropy).all()
    ids = torch.sort(x.double(), dim=-1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(r.top_ids, ids)
    lp = e.lp.gather(-1, ids)
    close(r.top_logprobs, lp.float().double(), e.lp_bound(lp), "top_logprobs")

    a, h = (torch.randn(rows, generator=g).to(DEV) for _ in range(2))
    got = esa.layer_ops.token_logprobs_backward(x, tokens, r, a, h)
    a, h = a.double()[:, None], h.double()[:, None]
    hot = torch.zeros(x.shape, dtype=torch.float64, device=DEV)
    hot[torch.arange(rows), tokens] = 1.0
    H = e.entropy[:, None]
    want = a * (hot - e.p) - h * e.p * (e.lp.masked_fill(e.p == 0, 0.0) + H)
    el = e.err_log[:, None] + 2 * U * e.log_s.abs()[:, None]
    ep = 3 * U * e.z.abs() + 5 * U + el
    size = a.abs() + h.abs() * (H + e.log_s[:, None] + e.z.abs())
    slack = (e.p * (size * (ep + 5 * U) + h.abs() * (e.err_entropy[:, None] + el))
             + U * hot * a.abs() + 2.0 ** -126)
    half_step = torch.finfo(dtype).eps / 2
    close(got, want, half_step * (want.abs() + slack) + slack + TINY[dtype], "dlogits")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [2, 30])
def test_logits_of_the_product_right_before(esa, dtype, rows):
    """The 4-bit LM head and the scores of its logits, issued back to back into the same
    memory: each call scores the logits of the product right before it."""
    lops = esa.layer_ops
    g = torch.Generator().manual_seed(rows)
    head = lops.quantize_weight4((0.2 * torch.randn(20000, 512, generator=g)).to(DEV, dtype))
    xs = [torch.randn(rows, 512, generator=g).to(DEV, dtype) for _ in range(12)]
    tokens = torch.randint(0, 20000, (rows,), generator=g).to(DEV)
    want = []
    for x in xs:
        y = lops.linear4(x, head)
        torch.cuda.synchronize()
        want.append(lops.token_logprobs(y, tokens, top_k=5))
        torch.cuda.synchronize()
        del y                                  # its memory serves the next product
    got = [lops.token_logprobs(lops.linear4(x, head), tokens, top_k=5) for x in xs]
    for a, b in zip(got, want):
        assert torch.equal(a.logprobs, b.logprobs) and torch.equal(a.entropy, b.entropy)
        assert torch.equal(a.top_ids, b.top_ids) and torch.equal(a.top_logprobs, b.top_logprobs)
