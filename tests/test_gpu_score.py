"""GPU: log probabilities of tokens, entropies, top alternatives and their gradient,
against plain formulas in float64.

Tolerances count roundings.  u = 2^-24 is float32's unit.  With z = x - m, p the
probabilities and S the sum of exp(z):
  z               one rounding: u |z|
  exp(z)          the product with log2(e) and that constant's own rounding move the
                  exponent by 2 u |z|, the hardware's exp2 is off by 4 u: 3 u |z| + 4 u
                  relative, the error of z included
  a sum of terms  a chain of at most n_add additions: n_add u relative, as no term is
                  negative
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


@pytest.fixture(scope="module")
def esa():
    import elastic_sparse_attention_b200 as mod
    return mod


def n_add(V):
    """Additions a term goes through: its thread's (64 threads at least share a row, an
    odd and an even chain each), then some 20 joins with two roundings each."""
    return V // 64 + 16 + 40


class Exact:
    def __init__(self, x, tokens):
        z = x.double()
        self.m = z.max(-1, keepdim=True).values
        self.lp = torch.log_softmax(z, -1)
        self.p = self.lp.exp()
        self.log_s = torch.logsumexp(z - self.m, -1)
        self.z = (z - self.m).masked_fill(self.p == 0, 0.0)
        plp = (self.p * self.lp).masked_fill(self.p == 0, 0.0)
        self.entropy = -plp.sum(-1)
        V = x.shape[-1]
        abs_z = (self.p * self.z.abs()).sum(-1)
        # relative error of S, then of ln S and of S1 / S
        self.err_s = U * (3 * abs_z + 4 + n_add(V))
        self.err_log = 1.01 * self.err_s + 2 * U * self.log_s.abs()
        second = (self.p * self.z * self.z).sum(-1)
        self.err_entropy = (self.err_log + U * (3 * second + (6 + n_add(V)) * abs_z)
                            + 1.01 * self.err_s * abs_z + 2 * U * (abs_z + self.entropy.abs()))
        t = tokens.clamp_min(0)[..., None]
        self.token_lp = self.lp.gather(-1, t)[..., 0]
        self.token_lp = self.token_lp.masked_fill(tokens == -100, 0.0)

    def lp_bound(self, lp):
        return self.err_log[..., None] + 3 * U * (lp.abs() + self.log_s.abs()[..., None])


def close(got, want, bound, what):
    assert got.shape == want.shape, what
    same = (got.double() == want) | (got.isnan() & want.isnan())
    bad = ~(same | ((got.double() - want).abs() <= bound))
    assert not bad.any(), (what, int(bad.sum()), got[bad][:4].tolist(), want[bad][:4].tolist())


def order(x):
    """Ids by value, NaN first, equal ones (-0 and 0 too) by ascending id."""
    key = torch.where(x.isnan(), math.inf, x.double())
    nan_first = torch.sort(x.isnan().int(), dim=-1, descending=True, stable=True).indices
    key = key.gather(-1, nan_first)
    # among equal keys NaNs lie before +infinity already
    return nan_first.gather(-1, torch.sort(key, dim=-1, descending=True, stable=True).indices)


def make(kind, rows, V, dtype, g):
    x = 3 * torch.randn(rows, V, generator=g)
    if kind == "masked":
        x[torch.rand(rows, V, generator=g) < 0.5] = -math.inf
        x[:, V // 2] = 1.0
    elif kind == "one left":
        x[:] = -math.inf
        x[torch.arange(rows), torch.randint(0, V, (rows,), generator=g)] = 0.5
    elif kind == "lowest":                  # a mask of the type's lowest value alone
        x[:] = torch.finfo(dtype).min
    elif kind == "lowest and infinite":
        x[:] = torch.finfo(dtype).min
        x[torch.rand(rows, V, generator=g) < 0.5] = -math.inf
        x[:, V // 2] = torch.finfo(dtype).min
    elif kind == "ties":
        x = x.round() / 2
        x[x.abs() < 0.3] = -0.0
    elif kind == "equal":
        x[:] = 1.25
    elif kind == "rising":
        x = torch.linspace(-9, 9, V).expand(rows, V).clone()
    elif kind == "far":                     # large offsets, one dominant logit
        x = x + 2000.0
        x[:, V // 3] += 30
    return x.to(DEV, dtype)


KINDS = ["normal", "masked", "one left", "lowest", "lowest and infinite", "ties", "equal", "rising",
         "far"]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,V,top", [
    (1, 1, 1), (3, 7, 7), (5, 8, 3), (2, 9, 0), (4, 33, 32), (7, 100, 20), (300, 513, 5),
    (2, 4097, 32), (1, 32000, 20), (40, 8192, 1), (160, 5000, 8), (9, 50021, 32), (1, 131075, 32)])
def test_forward(esa, dtype, kind, rows, V, top):
    g = torch.Generator().manual_seed(rows * V + top)
    x = make(kind, rows, V, dtype, g)
    tokens = torch.randint(0, V, (rows,), generator=g).to(DEV)
    if rows > 2:
        tokens[1] = -100
    want = Exact(x, tokens)
    esa.ops.device_errors()
    for ids in (tokens, tokens.to(torch.int32)):
        r = esa.layer_ops.token_logprobs(x, ids, top_k=top)
        close(r.logprobs, want.token_lp, want.lp_bound(want.token_lp[:, None])[:, 0], "logprobs")
        close(r.entropy, want.entropy, want.err_entropy, "entropy")
        close(r.logsumexp, want.m[:, 0] + want.log_s,
              want.err_log + U * (want.m[:, 0].abs() + want.log_s), "logsumexp")
        if top:
            first = order(x)[:, :top]
            assert torch.equal(r.top_ids, first)
            lp = want.lp.gather(-1, first)
            close(r.top_logprobs, lp, want.lp_bound(lp), "top_logprobs")
        else:
            assert r.top_ids is None and r.top_logprobs is None
    assert esa.ops.device_errors() == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_without_a_distribution(esa, dtype):
    """NaN, +infinity, -infinity alone; the alternatives are in order all the same."""
    g = torch.Generator().manual_seed(3)
    for V in (12, 700, 40000):
        x = torch.randn(6, V, generator=g)
        x[0, V // 2] = math.nan
        x[1, 5] = math.inf
        x[2] = -math.inf
        x[3, [1, V - 1]] = math.nan
        x[3, 0] = math.inf
        x[4, 1:] = -math.inf
        x = x.to(DEV, dtype)
        tokens = torch.full((6,), 3, device=DEV)
        top = 10
        r = esa.layer_ops.token_logprobs(x, tokens, top_k=top)
        nan = torch.tensor([True, True, True, True, False, False], device=DEV)
        assert torch.equal(r.logprobs.isnan(), nan) and torch.equal(r.entropy.isnan(), nan)
        assert r.logprobs[4] == -math.inf and r.entropy[4] == 0
        assert torch.equal(r.top_ids, order(x)[:, :top])
        assert r.top_logprobs[nan].isnan().all()
        assert r.top_logprobs[4, 0] == 0 and (r.top_logprobs[4, 1:] == -math.inf).all()
        # ignored rows have no gradient whatever they hold
        ignored = torch.full((6,), -100, device=DEV)
        s = esa.layer_ops.token_logprobs(x, ignored)
        assert not s.logprobs.any()
        d = esa.layer_ops.token_logprobs_backward(x, ignored, s, torch.ones(6, device=DEV))
        assert not d.any()


def test_tokens_outside_the_vocabulary(esa):
    bit = esa._lib.DEVERR_TOKEN_RANGE
    x = torch.randn(6, 300, device=DEV)
    tokens = torch.tensor([0, 300, -1, 299, 1 << 40, -100], device=DEV)
    esa.ops.device_errors()
    r = esa.layer_ops.token_logprobs(x, tokens)
    assert esa.ops.device_errors() == bit
    assert r.logprobs.isnan().tolist() == [False, True, True, False, True, False]
    assert not r.entropy.isnan().any()
    d = esa.layer_ops.token_logprobs_backward(x, tokens, r, torch.ones(6, device=DEV))
    assert esa.ops.device_errors() == bit
    assert d.isnan().any(-1).tolist() == [False, True, True, False, True, False]
    esa.layer_ops.token_logprobs(x, tokens[[0, 3, 5, 0, 3, 5]])
    assert esa.ops.device_errors() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset,V,stride", [(0, 1000, 1024), (1, 1000, 1024), (3, 777, 781),
                                             (5, 40001, 40007)])
def test_strided_rows(esa, dtype, offset, V, stride):
    """A slice of the columns of a padded buffer: rows begin at any element, what lies
    between them is neither read into the result nor written."""
    g = torch.Generator().manual_seed(V)
    buf = torch.full((5, stride), math.nan).to(DEV, dtype)
    x = buf[:, offset:offset + V]
    x.copy_(torch.randn(5, V, generator=g))
    tokens = torch.randint(0, V, (5,), generator=g).to(DEV)
    lops = esa.layer_ops
    a, b = lops.token_logprobs(x, tokens, top_k=4), lops.token_logprobs(x.contiguous(), tokens, top_k=4)
    want = Exact(x, tokens)
    close(a.logprobs, want.token_lp, want.lp_bound(want.token_lp[:, None])[:, 0], "logprobs")
    assert torch.equal(a.top_ids, b.top_ids)
    dlp, de = (torch.randn(5, generator=g).to(DEV) for _ in range(2))
    d = lops.token_logprobs_backward(x.contiguous(), tokens, a, dlp, de)
    out = torch.full((5, V + 3), 7.0, device=DEV, dtype=dtype)
    got = lops.token_logprobs_backward(x, tokens, a, dlp, de, out=out[:, 2:2 + V])
    assert torch.equal(got, d) and (out[:, :2] == 7).all() and (out[:, 2 + V:] == 7).all()
    keep = buf.clone()
    assert torch.equal(lops.token_logprobs_backward(x, tokens, a, dlp, de, out=x), d)     # in place
    pad = torch.ones(stride, dtype=torch.bool, device=DEV)
    pad[offset:offset + V] = False
    assert torch.equal(buf[:, pad].isnan(), keep[:, pad].isnan())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["normal", "masked", "one left", "lowest", "far"])
@pytest.mark.parametrize("rows,V", [(1, 1), (3, 7), (4, 100), (70, 513), (2, 32000), (5, 50021)])
@pytest.mark.parametrize("which", ["both", "logprobs", "entropy"])
def test_backward(esa, dtype, kind, rows, V, which):
    g = torch.Generator().manual_seed(rows + V)
    x = make(kind, rows, V, dtype, g)
    tokens = torch.randint(0, V, (rows,), generator=g).to(DEV)
    if rows > 2:
        tokens[1] = -100
    dlp = torch.randn(rows, generator=g).to(DEV) if which != "entropy" else None
    de = torch.randn(rows, generator=g).to(DEV) if which != "logprobs" else None
    r = esa.layer_ops.token_logprobs(x, tokens)
    got = esa.layer_ops.token_logprobs_backward(x, tokens, r, dlp, de)
    e = Exact(x, tokens)
    zero = torch.zeros(rows, 1, dtype=torch.float64, device=DEV)
    a = zero if dlp is None else dlp.double()[:, None].masked_fill((tokens == -100)[:, None], 0.0)
    h = zero if de is None else de.double()[:, None]
    hot = torch.zeros(x.shape, dtype=torch.float64, device=DEV)
    hot[torch.arange(rows), tokens.clamp_min(0)] = 1.0
    lp = e.lp.masked_fill(e.p == 0, 0.0)
    H = e.entropy[:, None]
    want = a * (hot - e.p) - h * e.p * (lp + H)
    # p: exponent moved by 3 u |z| + the error of ln S and two roundings of it; the
    # factor a + h (H - ln S) + h z: its roundings and the errors of H and ln S
    el = e.err_log[:, None] + 2 * U * e.log_s.abs()[:, None]
    ep = 3 * U * e.z.abs() + 5 * U + el
    size = a.abs() + h.abs() * (H + e.log_s[:, None] + e.z.abs())
    slack = (e.p * (size * (ep + 5 * U) + h.abs() * (e.err_entropy[:, None] + el))
             + U * hot * a.abs() + 2.0 ** -126)
    half_step = torch.finfo(dtype).eps / 2
    assert got.dtype == dtype
    close(got, want, half_step * (want.abs() + slack) + slack + TINY[dtype], "dlogits")


def test_gradient_is_the_difference_quotient(esa):
    """<dx, D> against (f(x + hD) - f(x - hD)) / 2h of f = <lp, a> + <H, b> in float64:
    the truncation is h^2 / 6 of the third derivative, below 1e-7 here."""
    g = torch.Generator().manual_seed(1)
    x, D = (torch.randn(20, 300, generator=g, dtype=torch.float64) for _ in range(2))
    x = x.float().double()
    tokens = torch.randint(0, 300, (20,), generator=g)
    a, b = (torch.randn(20, generator=g, dtype=torch.float64).float() for _ in range(2))

    def f(v):
        lp = torch.log_softmax(v, -1)
        return ((lp[torch.arange(20), tokens] * a).sum() - ((lp.exp() * lp).sum(-1) * b).sum())
    h = 1e-4
    quotient = (f(x + h * D) - f(x - h * D)) / (2 * h)
    xd = x.float().to(DEV)
    r = esa.layer_ops.token_logprobs(xd, tokens.to(DEV))
    d = esa.layer_ops.token_logprobs_backward(xd, tokens.to(DEV), r, a.to(DEV), b.to(DEV))
    terms = d.double().cpu() * D
    # each entry some 100 u of its own size (test_backward), the quotient 1e-16 / h
    assert abs(terms.sum() - quotient) <= 200 * U * terms.abs().sum() + 1e-6


def test_shapes_and_empty_calls(esa):
    lops = esa.layer_ops
    x = torch.randn(2, 3, 40, device=DEV)
    t = torch.randint(0, 40, (2, 3), device=DEV)
    r = lops.token_logprobs(x, t, top_k=2)
    assert r.logprobs.shape == (2, 3) and r.top_ids.shape == (2, 3, 2) and r.stats.shape == (2, 3, 2)
    one = lops.token_logprobs(x[0, 1], t[0, 1], top_k=2)          # a row by itself
    assert one.logprobs.shape == () and torch.equal(one.top_ids, r.top_ids[0, 1])
    none = lops.token_logprobs(x[:0], t[:0], top_k=3)
    assert none.top_ids.shape == (0, 3, 3)
    assert lops.token_logprobs_backward(x[:0], t[:0], none, none.logprobs).shape == (0, 3, 40)


def test_refusals(esa):
    lops = esa.layer_ops
    x = torch.randn(4, 50, device=DEV)
    t = torch.zeros(4, dtype=torch.int64, device=DEV)
    r = lops.token_logprobs(x, t)
    one = torch.ones(4, device=DEV)
    for bad, kw in ((ValueError, dict(top_k=33)), (ValueError, dict(top_k=-1))):
        with pytest.raises(bad):
            lops.token_logprobs(x, t, **kw)
    with pytest.raises(ValueError):
        lops.token_logprobs(x[:, :10], t, top_k=11)
    with pytest.raises(ValueError, match="tokens"):
        lops.token_logprobs(x, t[:3])
    with pytest.raises(TypeError):
        lops.token_logprobs(x, t.float())
    with pytest.raises(TypeError):
        lops.token_logprobs(x.double(), t)
    with pytest.raises(ValueError):
        lops.token_logprobs(x.t(), torch.zeros(50, dtype=torch.int64, device=DEV))
    with pytest.raises(ValueError):
        lops.token_logprobs(x[:1].expand(4, 50), t)               # rows on top of each other
    with pytest.raises(ValueError):
        lops.token_logprobs(x[:, :0], t)
    with pytest.raises(ValueError, match="dlogprobs"):
        lops.token_logprobs_backward(x, t, r, one[:3])
    with pytest.raises(ValueError, match="dentropy"):
        lops.token_logprobs_backward(x, t, r, one, one.double())
    with pytest.raises(ValueError, match="out"):
        lops.token_logprobs_backward(x, t, r, one, out=x[:3])
    with pytest.raises(ValueError, match="stats"):
        lops.token_logprobs_backward(x[:3], t[:3], r, one[:3])


def test_captured_and_on_another_stream(esa):
    lops = esa.layer_ops
    x = torch.randn(6, 9000, device=DEV, dtype=torch.bfloat16)
    t = torch.randint(0, 9000, (6,), device=DEV)
    one = torch.randn(6, device=DEV)

    def call():
        r = lops.token_logprobs(x, t, top_k=7)
        return r, lops.token_logprobs_backward(x, t, r, one, one)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r, d = call()
    for seed in (1, 2):
        x.copy_(torch.randn(6, 9000, generator=torch.Generator().manual_seed(seed)))
        t.copy_(torch.randint(0, 9000, (6,), generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        want, wd = call()
        assert torch.equal(r.logprobs, want.logprobs) and torch.equal(r.top_ids, want.top_ids)
        assert torch.equal(d, wd) and torch.equal(r.entropy, want.entropy)
    # two streams at once, each its own rows
    streams = [torch.cuda.Stream() for _ in range(2)]
    big = [torch.randn(64, 32000, device=DEV) for _ in range(2)]
    tok = torch.randint(0, 32000, (64,), device=DEV)
    wants = [lops.token_logprobs(b, tok, top_k=20) for b in big]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                outs[i].append(lops.token_logprobs(big[i], tok, top_k=20))
    torch.cuda.synchronize()
    for want, got in zip(wants, outs):
        for o in got:
            assert torch.equal(o.top_ids, want.top_ids) and torch.equal(o.logprobs, want.logprobs)


# ---------------------------------------------------------------------------
# the decoder stack's differentiable scores
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("chunk", [1000, 70])
def test_stack_token_logprobs(esa, chunk):
    """Values and all gradients against log_softmax of the whole logits (float32)."""
    stack = esa.ElasticDecoderStack(vocab_size=301, hidden_size=128, num_hidden_layers=2,
                                    num_attention_heads=4, num_key_value_heads=2, head_dim=32,
                                    intermediate_size=192, attention_length=16, max_seq_len=256,
                                    dtype=torch.float32, device=DEV, loss_chunk_rows=chunk)
    g = torch.Generator().manual_seed(0)
    ids = torch.randint(0, 301, (2, 90), generator=g).to(DEV)
    labels = ids.clone()
    labels[0, 10:20] = -100
    wl, we = (torch.randn(2, 90, generator=g).to(DEV) for _ in range(2))

    def grads(use_entropy):
        lp, ent = stack.token_logprobs(ids, labels)
        loss = (lp * wl).sum() + ((ent * we).sum() if use_entropy else 0)
        return lp, ent, torch.autograd.grad(loss, list(stack.parameters()))

    def reference(use_entropy):
        y = stack(ids)
        lsm = torch.log_softmax(y.float() @ stack.lm_head.float().t(), -1)
        nxt = torch.full_like(labels, -100)
        nxt[:, :-1] = labels[:, 1:]
        lp = lsm.gather(-1, nxt.clamp_min(0)[..., None])[..., 0] * (nxt != -100)
        ent = -(lsm.exp() * lsm).sum(-1)
        loss = (lp * wl).sum() + ((ent * we).sum() if use_entropy else 0)
        return lp, ent, torch.autograd.grad(loss, list(stack.parameters()))
    for use in (True, False):
        (lp, ent, gr), (rlp, rent, rgr) = grads(use), reference(use)
        assert (lp[:, -1] == 0).all() and (lp[0, 9:19] == 0).all()
        assert (lp - rlp).abs().max() <= 1e-4 and (ent - rent).abs().max() <= 1e-4
        for (name, _), a, b in zip(stack.named_parameters(), gr, rgr):
            assert (a - b).abs().max() <= 1e-3 * b.abs().max() + 1e-7, name
    lp, ent = stack.token_logprobs(ids)
    (g1,) = torch.autograd.grad(ent.sum(), [stack.lm_head], create_graph=True)
    with pytest.raises(RuntimeError, match="second derivatives"):
        g1.sum().backward()


def test_stack_scores_captured(esa):
    """A forward and backward captured into a graph and replayed (torch wants no eager
    graph of the same parameters alive at the capture)."""
    stack = esa.ElasticDecoderStack(vocab_size=200, hidden_size=64, num_hidden_layers=1,
                                    num_attention_heads=2, head_dim=32, intermediate_size=96,
                                    attention_length=8, max_seq_len=64, dtype=torch.float32,
                                    device=DEV)
    ids = torch.randint(0, 200, (2, 20), device=DEV)
    params = list(stack.parameters())

    def step():
        lp, ent = stack.token_logprobs(ids)
        return [t.clone() for t in torch.autograd.grad(lp.sum() + 0.1 * ent.sum(), params)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (1, 2):
        ids.copy_(torch.randint(0, 200, (2, 20), generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)
