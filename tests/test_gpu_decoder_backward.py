"""GPU: what the decoder stack's backward pass takes from the forward pass it
belongs to, whatever happens to the stack in between, and what it holds while
it runs."""
import pytest
import torch

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
