"""Shapes that the row operators refuse, and how: a ValueError that names the
operand's fault, not an error of the arithmetic on its shape."""
import pytest
import torch

DEV = "cuda:0"


def test_rows_without_elements_or_axes(esa):
    lops = esa.layer_ops
    with pytest.raises(ValueError, match="at least one element"):
        lops._rows(torch.empty(3, 0), 0)
    with pytest.raises(ValueError, match="feature axis"):
        lops._shape(torch.empty(()))
    assert lops._rows(torch.empty(0, 8), 8) == 0 and lops._rows(torch.empty(2, 3, 8), 8) == 6
    packed = lops.PackedRows(torch.empty((), dtype=torch.uint8), torch.empty(()), "int8",
                             torch.float32)
    with pytest.raises(ValueError, match="feature axis"):
        lops._check_packed(packed)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(3, 0), (0, 0), ()])
def test_operators_refuse_such_rows(esa, shape):
    lops = esa.layer_ops
    x = torch.empty(shape, device=DEV)
    w = torch.empty(shape[-1:], device=DEV)
    packed = lops.PackedRows(x.to(torch.uint8), x.new_empty(shape[:-1] + (0,)), "int8",
                             torch.float32)
    for call in (lambda: lops.quantize_rows(x), lambda: lops.rmsnorm_forward_packed(x, w, 1e-6),
                 lambda: lops.swiglu_forward_packed(x), lambda: lops.dequantize_rows(packed),
                 lambda: lops.rmsnorm_from_packed(packed, w, 1e-6)):
        with pytest.raises(ValueError):
            call()


def test_rotation_tables_of_another_kind(esa):
    """A stack cast with ``.half()`` has a half table, which the kernels would read
    as float32, past its end."""
    check = esa.layer_ops._check_inv_freq
    table = esa.layer_ops.rope_inv_freq(64, 10000.0, "cpu")
    check(table, 64)
    for bad in (table.half(), table[:16], table.repeat(2)[::2], table.double()):
        with pytest.raises(ValueError, match="inv_freq"):
            check(bad, 64)


@pytest.mark.gpu
def test_rope_refuses_such_tables(esa):
    q = torch.randn(1, 2, 3, 64, device=DEV)
    inv = esa.layer_ops.rope_inv_freq(64, 10000.0, DEV)
    for bad in (inv.half(), inv[:16]):
        with pytest.raises(ValueError, match="inv_freq"):
            esa.layer_ops.rope_(q, None, bad)
