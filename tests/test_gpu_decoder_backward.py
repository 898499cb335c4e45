"""GPU: what the decoder stack's backward pass takes from the forward pass it
belongs to, whatever happens to the stack in between, and what it holds while
it runs."""
import pytest
import torch
import torch.utils.checkpoint

from test_gpu_decoder_options import CFG, build

pytestmark = pytest.mark.gpu

CKPT8 = dict(activation_checkpointing=True, activation_storage="int8")


def gradients(m):
    return {n: p.grad.clone() for n, p in m.named_parameters()}


@pytest.mark.parametrize("kw", [CKPT8, dict(activation_storage="int8")],
                         ids=["checkpoints", "gate_up"])
def test_options_set_after_the_forward_pass_do_not_reach_its_backward(kw):
    """The 8-bit rows are read in the format they were written in."""
    want = None
    for storage, checkpointing in ((None, None), ("e4m3", None), ("int8", False), ("int8", True)):
        m, ids = build(qk_norm=True, **kw)
        loss = m(ids, labels=ids)
        if storage is not None:
            m.activation_storage = storage
        if checkpointing is not None:
            m.checkpointing = checkpointing
        loss.backward()
        got = gradients(m)
        want = want or got
        for n in want:
            assert torch.equal(got[n], want[n]), (n, storage, checkpointing)


def test_functional_call_with_8_bit_checkpoints():
    """Weights that the stack has only during the call: the backward runs the
    layers with them again."""
    m, ids = build(qk_norm=True, **CKPT8)
    g = torch.Generator().manual_seed(9)
    other = {n: (p.detach() + 0.01 * torch.randn(p.shape, generator=g).to(p.device)).requires_grad_()
             for n, p in m.named_parameters()}
    loss = torch.func.functional_call(m, other, (ids,), dict(labels=ids))
    loss.backward()
    assert all(p.grad is None for p in m.parameters())
    with torch.no_grad():
        for n, p in m.named_parameters():
            p.copy_(other[n])
    want = m(ids, labels=ids)
    want.backward()
    assert torch.equal(loss, want)
    for n, grad in gradients(m).items():
        assert torch.equal(other[n].grad, grad), n


@pytest.mark.parametrize("nl", [2, 4])
def test_8_bit_checkpoints_lower_the_peak_of_a_step(nl):
    """Where a row per token is the unit (8 MiB here, the weights 15 MiB a layer),
    the whole step's peak stays below the one of checkpoints that keep two full
    rows per layer, from two layers on."""
    cfg = dict(CFG, d=512, F=1024, nl=nl, L=8192, B=1, chunk=512)

    def peak(**kw):
        m, ids = build(torch.bfloat16, cfg, **kw)
        m(ids, labels=ids).backward()      # the key plans and gradients are there
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        m(ids, labels=ids).backward()
        return torch.cuda.max_memory_allocated() - before

    full, packed = peak(activation_checkpointing=True), peak(**CKPT8)
    assert packed < full, (packed, full)


def test_8_bit_checkpoints_backward_twice():
    """A graph that is kept runs again; a backward that stops at the last norm
    leaves nothing behind that a later one takes for its own."""
    m, ids = build(qk_norm=True, **CKPT8)
    m(ids, labels=ids).backward()
    want = gradients(m)
    m.zero_grad(set_to_none=True)
    loss = m(ids, labels=ids)
    dw, = torch.autograd.grad(loss, m.final_norm, retain_graph=True)
    assert torch.equal(dw, want["final_norm"])
    loss.backward(retain_graph=True)
    for n, grad in gradients(m).items():
        assert torch.equal(grad, want[n]), n
    m.zero_grad(set_to_none=True)
    loss.backward()
    for n, grad in gradients(m).items():
        assert torch.equal(grad, want[n]), n


def test_8_bit_checkpoints_of_hidden_states():
    """Without labels: the last layer's residual sum takes no gradient."""
    m, ids = build(**CKPT8)
    y = m(ids)
    g = torch.Generator().manual_seed(3)
    c = torch.randn(y.shape, generator=g).to(y.device)
    (y * c).sum().backward()
    want, ids = build(activation_checkpointing=True)
    (want(ids) * c).sum().backward()
    for (n, p), q in zip(m.named_parameters(), want.parameters()):
        if n == "lm_head":
            assert p.grad is None
            continue
        # gradients at inputs off by at most 1/254 of their group's largest
        assert torch.nn.functional.cosine_similarity(p.grad.flatten(), q.grad.flatten(), 0) > 0.99


def test_captured_step_with_8_bit_checkpoints():
    """A step captured in a graph, an eager step of the same stack before and
    between its replays."""
    m, ids = build(**CKPT8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            m.zero_grad(set_to_none=True)
            m(ids, labels=ids).backward()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    want = gradients(m)
    m.zero_grad(set_to_none=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m(ids, labels=ids).backward()
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        for n, grad in gradients(m).items():
            assert torch.equal(grad, want[n]), n


@pytest.mark.parametrize("kw", [{}, dict(embed_scale=2.0), dict(qk_norm=True),
                                dict(activation_storage="int8"), CKPT8],
                         ids=lambda kw: "-".join(kw) or "plain")
@pytest.mark.parametrize("of", ["embed", "layers.0.down_proj", "final_norm", "lm_head"])
def test_second_derivatives_are_refused(kw, of):
    """The kernels have none; a graph of the gradient would lack their part."""
    m, ids = build(**kw)
    p = dict(m.named_parameters())[of]
    want, = torch.autograd.grad(m(ids, labels=ids), p)
    got, = torch.autograd.grad(m(ids, labels=ids), p, create_graph=True)
    assert torch.equal(got, want)
    with pytest.raises(RuntimeError, match="no second derivatives"):
        got.square().sum().backward()


@pytest.mark.parametrize("bad", [-1, CFG["V"], 1 << 40])
@pytest.mark.parametrize("kw", [{}, CKPT8], ids=["kept", "checkpoints"])
def test_a_token_outside_the_vocabulary_shows_in_the_loss(kw, bad):
    """With the library's lookup such a token is no device assert, but no silent
    zero row either (the labels here are valid)."""
    import elastic_sparse_attention_b200 as esa
    m, ids = build(embed_scale=2.0, padding_idx=0, **kw)
    esa.ops.device_errors()
    clean = m(ids, labels=ids)
    assert clean.isfinite() and esa.ops.device_errors() == 0
    wrong = ids.clone()
    wrong[1, 7] = bad
    hidden = m(wrong)
    assert hidden[1, 7].isnan().all() and hidden[0].isfinite().all()
    loss = m(wrong, labels=ids)
    assert loss.isnan()
    loss.backward()
    assert not m.layers[0].qkv_proj.grad.isfinite().all()
    assert esa.ops.device_errors() == esa._lib.DEVERR_TOKEN_RANGE


def test_8_bit_checkpoints_keep_no_run_that_nothing_differentiates():
    """Only the last norm's weight takes a gradient: the layer runs again for its
    input, and nothing of that run outlives the backward."""
    m, ids = build(**CKPT8)
    for p in m.parameters():
        p.requires_grad_(p is m.final_norm)
    want, _ = build(activation_checkpointing=True)
    want(ids, labels=ids).backward()
    m(ids, labels=ids).backward()
    assert torch.nn.functional.cosine_similarity(m.final_norm.grad, want.final_norm.grad, 0) > 0.99
    loss = m(ids, labels=ids)
    held = torch.cuda.memory_allocated()
    loss.backward()
    assert torch.cuda.memory_allocated() <= held
    # the same where all may take gradients, but the call asks for one alone
    m, ids = build(**CKPT8)
    loss = m(ids, labels=ids)
    held = torch.cuda.memory_allocated()
    torch.autograd.grad(loss, m.final_norm)
    assert torch.cuda.memory_allocated() <= held


def test_8_bit_checkpoints_inside_other_savers():
    """Saved tensors that a hook moves to the host, and the whole stack inside a
    checkpoint of the caller's: the layers' weights are still the ones that get
    the gradients."""
    m, ids = build(qk_norm=True, embed_scale=2.0, **CKPT8)
    m(ids, labels=ids).backward()
    want = gradients(m)
    m.zero_grad(set_to_none=True)
    with torch.autograd.graph.save_on_cpu():
        loss = m(ids, labels=ids)
    loss.backward()
    for n, grad in gradients(m).items():
        assert torch.equal(grad, want[n]), n
    m.zero_grad(set_to_none=True)
    torch.utils.checkpoint.checkpoint(lambda: m(ids, labels=ids), use_reentrant=False).backward()
    for n, grad in gradients(m).items():
        assert torch.equal(grad, want[n]), n
