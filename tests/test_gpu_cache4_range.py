"""GPU: the 4-bit key / value cache at the ends of its range."""
import pytest
import torch

from test_gpu_cache4 import DEV, decoded, head_rows

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def esa():
    import elastic_sparse_attention_b200 as mod
    return mod


@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("S,L", [(10, 25), (10, 10), (1, 300), (70, 1000)])
def test_more_rows_than_the_cache_has_positions(esa, D, S, L):
    """Row l is position start + l, and only positions of the cache are written or
    read, however far outside the call begins."""
    starts = [0, 1, S - 1, S, S + 1, 1 << 62, -1, -(S - 1), -S, -(S + 1), -(S + 5), -(L - 1), -L,
              -(L + 1), -(L + S), -(1 << 24), -(1 << 40), -(1 << 62)]
    B = len(starts)
    g = torch.Generator().manual_seed(S + L)
    old, new = head_rows((B, 2, S, D), g, torch.float32), head_rows((B, 2, L, D), g, torch.float32)
    start = torch.tensor(starts, device=DEV)
    for counts in (None, torch.full((B,), L - L // 3)):
        n = L if counts is None else int(counts[0])
        cache = esa.PackedKVCache(B, 2, S, D, device=DEV)
        cache.write(old, old, 0)
        esa.ops.device_errors()
        cache.write(new, new, start, None if counts is None else counts.to(DEV))
        assert esa.ops.device_errors() == esa._lib.DEVERR_KV_RANGE
        want = decoded(old)
        fresh = decoded(new)
        for b, s in enumerate(starts):
            for p in range(max(s, 0), min(s + n, S)):
                want[b, :, p] = fresh[b, :, p - s]
        for t in cache.read(0, S, torch.float32):
            assert torch.equal(t.double(), want)
        out = torch.zeros(B, 2, L, D, dtype=torch.float64, device=DEV)
        for b, s in enumerate(starts):
            for p in range(max(s, 0), min(s + L, S)):
                out[b, :, p - s] = want[b, :, p]
        assert esa.ops.device_errors() == 0
        for t in cache.read(start, L, torch.float32):
            assert torch.equal(t.double(), out)
        assert esa.ops.device_errors() == esa._lib.DEVERR_KV_RANGE
