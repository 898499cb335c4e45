"""GPU: the serving session (4-bit projections, 4-bit caches, scores) as a run of its
operators: against a plain-torch restatement, prompts against single tokens, padded
batches, a captured step.

The restatement is given the keys and values that the session stored: its own differ
from the session's by float32 roundings, and where such a difference lies across the
border between two codes they would store values a whole step apart.  Each stored
value is checked against the restatement's: within half a step of the format (a
group's largest magnitude / 14, its bfloat16 step up to 2^-8 larger) and the 1e-4 by
which the activations may differ.
"""
import math

import pytest
import torch
import torch.nn.functional as F

from decoder_reference import rmsnorm, rope, swiglu
from oracle import naive, pattern

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.fixture(scope="module")
def esa():
    import elastic_sparse_attention_b200 as mod
    return mod


def make_stack(esa, dtype=torch.float32, **kw):
    args = dict(vocab_size=301, hidden_size=256, num_hidden_layers=3, num_attention_heads=4,
                num_key_value_heads=2, head_dim=64, intermediate_size=384, attention_length=16,
                max_seq_len=512, dtype=dtype, device=DEV)
    args.update(kw)
    stack = esa.ElasticDecoderStack(**args)
    with torch.no_grad():
        for p in stack.parameters():
            if p.dim() == 2:
                p.mul_(3)              # attention that is not flat
            elif p.numel() < 1000:
                p.add_(0.1 * torch.randn(p.shape, device=DEV).to(dtype))
    return stack


def reference(esa, stack, session, ids):
    """(hidden states, logits) in float32 of a whole prompt, with the decoded weights and the
    session's stored keys and values."""
    deq = lambda w: esa.layer_ops.dequantize_weight4(w, torch.float32)
    B, L = ids.shape
    Hq, Hkv, D = stack.Hq, stack.Hkv, stack.D
    positions = torch.arange(L, device=DEV)
    h = F.embedding(ids, stack.embed) * (stack.embed_scale or 1.0)
    for i, packed in enumerate(session.layers):
        wqkv, wo, wgu, wd = (deq(w) for w in packed)
        lw = stack.layers[i]
        x = (rmsnorm(h, lw.input_norm, stack.eps) @ wqkv.t()).view(B, L, Hq + 2 * Hkv, D)
        q, k, v = (t.transpose(1, 2) for t in x.split([Hq, Hkv, Hkv], 2))
        if lw.q_norm is not None:
            q, k = rmsnorm(q, lw.q_norm, stack.eps), rmsnorm(k, lw.k_norm, stack.eps)
        q, k = rope(q, positions, stack.inv_freq), rope(k, positions, stack.inv_freq)
        stored = session.caches[i].read(0, L, torch.float32)
        for own, kept in zip((k, v), stored):
            g = own.unflatten(-1, (-1, 32))
            half = (g.abs().amax(-1, keepdim=True) / 14 * (1 + 2.0 ** -8)).expand(g.shape).flatten(-2)
            assert ((own - kept).abs() <= half + 1e-4).all()
        idx, mask, _ = pattern.prepared_indices(Hq, stack.specs[i].attention_length, i,
                                                len(stack.layers), L, L, L)
        o, _ = naive.naive_forward(q, *stored, torch.from_numpy(idx).to(DEV),
                                   torch.from_numpy(mask).to(DEV), D ** -0.5, Hq // Hkv)
        h = h + o.transpose(1, 2).reshape(B, L, Hq * D) @ wo.t()
        h = h + swiglu(rmsnorm(h, lw.post_attention_norm, stack.eps) @ wgu.t()) @ wd.t()
    y = rmsnorm(h, stack.final_norm, stack.eps)
    return y, y @ deq(session.lm_head).t()


@pytest.mark.parametrize("qk_norm", [False, True])
@pytest.mark.parametrize("group,L", [(128, 100), (32, 20)])
@torch.no_grad()
def test_a_prompt_against_plain_torch(esa, qk_norm, group, L):
    torch.manual_seed(0)
    stack = make_stack(esa, qk_norm=qk_norm, embed_scale=4.0)
    session = esa.PackedDecoder(stack, 2, 300, group)
    ids = torch.randint(0, 301, (2, L), device=DEV)
    esa.ops.device_errors()
    scores = session.score(ids, top_k=6)
    y, logits = reference(esa, stack, session, ids)
    # as for the stack: float32 within 1e-4, here of values of order one
    lsm = torch.log_softmax(logits, -1)
    want = lsm[:, :-1].gather(-1, ids[:, 1:, None])[..., 0]
    assert (scores.logprobs[:, :-1] - want).abs().max() <= 2e-3 and not scores.logprobs[:, -1].any()
    assert (scores.entropy + (lsm.exp() * lsm).sum(-1)).abs().max() <= 2e-3
    top = lsm.gather(-1, scores.top_ids)
    assert (top - scores.top_logprobs).abs().max() <= 2e-3
    assert (lsm.topk(6).values - top).abs().max() <= 4e-3
    assert session.lengths.tolist() == [L, L] and esa.ops.device_errors() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@torch.no_grad()
def test_tokens_one_by_one_and_padded_batches(esa, dtype):
    """A prompt at once, in ragged padded pieces, token by token.  In float32 the scores
    agree within the activations' roundings.  In bfloat16 each run rounds its
    activations in places of its own: each is as far from the float32 run of the same
    weights as the others (twice the root mean square at most)."""
    torch.manual_seed(1)
    stack = make_stack(esa, dtype)
    exact = make_stack(esa)
    for p, q in zip(exact.parameters(), stack.parameters()):
        p.copy_(q)
    B, L = 3, 90
    ids = torch.randint(0, 301, (B, L), device=DEV)
    whole = esa.PackedDecoder(stack, B, L)
    a = whole.score(ids, top_k=4)
    pieces = esa.PackedDecoder(stack, B, L)
    fed = [0, 0, 0]
    lp, ent = a.logprobs.clone(), torch.zeros(B, L, device=DEV)
    for counts in ([40, 70, 10], [1, 0, 3], [30, 20, 77], [19, 0, 0]):
        n = max(counts)
        part = torch.zeros(B, n, dtype=torch.int64, device=DEV)
        for b, c in enumerate(counts):
            part[b, :c] = ids[b, fed[b]:fed[b] + c]
        r = pieces.score(part, torch.tensor(counts), top_k=4)
        for b, c in enumerate(counts):
            ent[b, fed[b]:fed[b] + c] = r.entropy[b, :c]
            if c:                           # a piece's last token has no next one
                assert r.logprobs[b, c - 1] == 0
                lp[b, fed[b]:fed[b] + c - 1] = r.logprobs[b, :c - 1]
            fed[b] += c
    assert fed == [L] * B and pieces.lengths.tolist() == fed
    single = esa.PackedDecoder(stack, B, L)
    one = torch.stack([single.score(ids[:, t:t + 1]).entropy[:, 0] for t in range(L)], 1)
    if dtype == torch.float32:
        for x, y in ((lp, a.logprobs), (ent, a.entropy), (one, a.entropy)):
            assert (x - y).abs().max() <= 1e-3
    else:
        e = esa.PackedDecoder(exact, B, L).score(ids)
        rms = lambda x, y: (x - y).square().mean().sqrt()
        assert rms(lp, e.logprobs) <= 2 * rms(a.logprobs, e.logprobs)
        assert rms(ent, e.entropy) <= 2 * rms(a.entropy, e.entropy)
        assert rms(one, e.entropy) <= 2 * rms(a.entropy, e.entropy)
    assert esa.ops.device_errors() == 0


@torch.no_grad()
def test_captured_decoding(esa):
    """One captured step, replayed: greedy decoding from the alternatives."""
    torch.manual_seed(2)
    stack = make_stack(esa, torch.bfloat16, qk_norm=True)
    prompt = torch.randint(0, 301, (2, 33), device=DEV)
    eager, graphed = (esa.PackedDecoder(stack, 2, 64) for _ in range(2))
    tok = [s.score(prompt, top_k=3).top_ids[:, -1:, 0].clone() for s in (eager, graphed)]
    assert torch.equal(*tok)
    ids = tok[1].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graphed.score(ids, torch.zeros(2, dtype=torch.int64, device=DEV), top_k=3)   # warm up
    torch.cuda.current_stream().wait_stream(side)
    assert graphed.lengths.tolist() == [33, 33]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = graphed.score(ids, top_k=3)
    for _ in range(10):
        graph.replay()
        w = eager.score(tok[0], top_k=3)
        assert torch.equal(r.top_ids, w.top_ids) and torch.equal(r.top_logprobs, w.top_logprobs)
        tok[0] = w.top_ids[:, :, 0]
        ids.copy_(r.top_ids[:, :, 0])
    assert graphed.lengths.tolist() == [43, 43] and esa.ops.device_errors() == 0


@torch.no_grad()
def test_limits_and_refusals(esa):
    stack = make_stack(esa)
    s = esa.PackedDecoder(stack, 2, 10)
    assert s.step(torch.zeros(2, 0, dtype=torch.int64, device=DEV)).shape == (2, 0, 256)
    assert s.score(torch.zeros(2, 0, dtype=torch.int64, device=DEV), top_k=2).top_ids.shape == (2, 0, 2)
    esa.ops.device_errors()
    ids = torch.randint(0, 301, (2, 12), device=DEV)
    y = s.step(ids)
    assert esa.ops.device_errors() == (esa._lib.DEVERR_KV_RANGE | esa._lib.DEVERR_QUERY_RANGE)
    t = esa.PackedDecoder(stack, 2, 12)
    assert torch.equal(t.step(ids)[:, :10], y[:, :10])       # those within are as ever
    s.reset()
    assert torch.equal(s.step(ids[:, :10]), t_first(esa, stack, ids))
    for bad in (ids[:1], ids[0]):
        with pytest.raises(ValueError):
            s.step(bad)
    with pytest.raises(ValueError, match="counts"):
        s.step(ids, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError, match="max_len"):
        esa.PackedDecoder(stack, 1, 513)
    with pytest.raises(ValueError, match="head_dim"):
        esa.PackedDecoder(make_stack(esa, head_dim=32), 1, 10)
    with pytest.raises(ValueError, match="top_k"):
        s.score(ids[:, :1], top_k=40)
    esa.ops.device_errors()
    dense = sum(p.numel() * 2 for p in stack.parameters() if p.dim() == 2)
    assert s.nbytes() - sum(c.nbytes() for c in s.caches) < dense / 3


def t_first(esa, stack, ids):
    return esa.PackedDecoder(stack, 2, 10).step(ids[:, :10])


@pytest.mark.parametrize("pad", [-100, 1 << 40])
@torch.no_grad()
def test_padding_with_any_id(esa, pad):
    """The rows of tokens are as with padding of an id of the vocabulary, with the
    library's lookup and with torch's."""
    torch.manual_seed(3)
    for kw in (dict(), dict(embed_scale=2.0)):
        stack = make_stack(esa, **kw)
        ids = torch.randint(0, 301, (3, 20), device=DEV)
        counts = torch.tensor([20, 7, 0], device=DEV)
        esa.ops.device_errors()
        a, b = (esa.PackedDecoder(stack, 3, 40) for _ in range(2))
        want = a.score(ids, counts, top_k=3)
        padded = ids.masked_fill(torch.arange(20, device=DEV) >= counts[:, None], pad)
        got = b.score(padded, counts, top_k=3)
        for i, n in enumerate(counts.tolist()):
            assert torch.equal(got.logprobs[i, :n], want.logprobs[i, :n])
            assert torch.equal(got.top_ids[i, :n], want.top_ids[i, :n])
        assert all(torch.equal(x.codes, y.codes) for x, y in zip(a.caches, b.caches))
        assert esa.ops.device_errors() == 0


@torch.no_grad()
def test_no_sequences_narrow_ids_and_small_chunks(esa):
    torch.manual_seed(4)
    stack = make_stack(esa)
    none = esa.PackedDecoder(stack, 0, 10)
    ids = torch.randint(0, 301, (2, 30), device=DEV)
    assert none.step(ids[:0]).shape == (0, 30, 256)
    r = none.score(ids[:0], top_k=2)
    assert r.logprobs.shape == (0, 30) and r.top_ids.shape == (0, 30, 2) and none.nbytes() > 0
    a, b, c = (esa.PackedDecoder(stack, 2, 40) for _ in range(3))
    counts = torch.tensor([30, 11], dtype=torch.int32)
    want = a.score(ids, counts.to(DEV).long(), top_k=3)
    got = b.score(ids.int(), counts, top_k=3)
    # (float32 products of few rows and of many sum in other orders)
    stack.loss_chunk_rows = 7
    parts = c.score(ids, counts, top_k=3)
    for i, n in enumerate(counts.tolist()):
        assert torch.equal(got.logprobs[i, :n], want.logprobs[i, :n])
        assert torch.equal(got.top_ids[i, :n], want.top_ids[i, :n])
        assert (parts.logprobs[i, :n] - want.logprobs[i, :n]).abs().max() <= 1e-3
        assert (parts.entropy[i, :n] - want.entropy[i, :n]).abs().max() <= 1e-3
    assert a.lengths.tolist() == b.lengths.tolist() == c.lengths.tolist() == [30, 11]


@torch.no_grad()
def test_half_precision_session(esa):
    """float16, prompts above and below the rows that are multiplied by codes: as far from
    the float32 run of the same weights as each other (twice the root mean square)."""
    torch.manual_seed(5)
    stack = make_stack(esa, torch.float16)
    exact = make_stack(esa)
    for p, q in zip(exact.parameters(), stack.parameters()):
        p.copy_(q)
    ids = torch.randint(0, 301, (1, 90), device=DEV)
    e = esa.PackedDecoder(exact, 1, 90).score(ids)
    whole = esa.PackedDecoder(stack, 1, 90).score(ids)
    s = esa.PackedDecoder(stack, 1, 90)
    parts = [s.score(ids[:, i:i + 30]).entropy for i in (0, 30, 60)]
    rms = lambda x, y: (x - y).square().mean().sqrt()
    assert rms(torch.cat(parts, 1), e.entropy) <= 2 * rms(whole.entropy, e.entropy)
    assert esa.ops.device_errors() == 0
