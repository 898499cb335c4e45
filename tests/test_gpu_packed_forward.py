"""GPU: the forward pass with activations kept in 8 bits against the one without.

h is the same bit for bit: one addition, one rounding.  The norm's and SwiGLU's
float32 arithmetic is not (sums in another order; for 16-bit types the
hardware's exponential and reciprocal), so a result may be rounded to the
neighbouring value of its type: at most one step apart, half a step on each
side, besides the float32 errors of the two.
"""
import pytest
import torch

from test_gpu_decoder_options import build

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def lops():
    import elastic_sparse_attention_b200 as esa
    return esa.layer_ops


def near(a, b, slack):
    """At most a step of the type apart, and the float32 errors ``slack`` (relative)
    of the two before their rounding."""
    assert a.dtype == b.dtype
    x, y = a.double(), b.double()
    top = torch.maximum(x.abs(), y.abs())
    tiny = torch.finfo(a.dtype).smallest_normal * torch.finfo(a.dtype).eps
    bound = (torch.finfo(a.dtype).eps + 2 * slack) * (1 + 2 * slack) * top + tiny
    assert ((x - y).abs() <= bound).all()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,dim", [(300, 256), (77, 1032), (64, 4096)])
def test_norm(lops, dtype, fmt, rows, dim):
    g = torch.Generator().manual_seed(dim)
    x, r = (torch.randn(rows, dim, generator=g).to(DEV, dtype) for _ in range(2))
    w = (1 + 0.1 * torch.randn(dim, generator=g)).to(DEV, dtype)
    h, y, rstd = lops.rmsnorm_forward(x, w, 1e-6, residual=r)
    h8, y8, rstd8, _ = lops.rmsnorm_forward_packed(x, w, 1e-6, residual=r, format=fmt)
    assert torch.equal(h, h8)
    # sums of at most dim / 32 + 6 squares in a row, halved by the root; mean, eps, root 5 u
    slack = ((max(dim / 32, 8) + 6) / 2 + 5) * U
    near(rstd, rstd8, slack)
    near(y, y8, slack + 2 * U)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,ffn", [(300, 384), (33, 1000), (40, 11008)])
def test_swiglu(lops, dtype, fmt, rows, ffn):
    g = torch.Generator().manual_seed(ffn)
    gu = (3 * torch.randn(rows, 2 * ffn, generator=g)).to(DEV, dtype)
    # |g| < 20: the exponential 2 u (hardware: 4 u + |g| u of its argument), 1 + e, the
    # reciprocal or quotient 2 u, two products: below 32 u
    assert gu.abs().max() < 20
    near(lops.swiglu_forward(gu), lops.swiglu_forward_packed(gu, fmt)[0], 32 * U)


@pytest.mark.parametrize("dtype,most", [(torch.float32, 1e-4), (torch.bfloat16, 2e-2)])
@pytest.mark.parametrize("ckpt", [False, True])
def test_hidden_states_of_a_training_step(dtype, most, ckpt):
    """The paths that a backward follows (``no_grad`` takes the unpacked one)."""
    m, ids = build(dtype, qk_norm=True, activation_checkpointing=ckpt)
    want = m(ids).float()
    for fmt in ("int8", "e4m3"):
        n, _ = build(dtype, qk_norm=True, activation_checkpointing=ckpt, activation_storage=fmt)
        got = n(ids).float()
        assert got.requires_grad
        assert (got - want).norm() <= most * want.norm()
