"""GPU: weights in 4 bits and products with them at the ends of their types' range."""
import pytest
import torch

from test_gpu_weight4 import DEV

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
