"""CPU: the layer entry points' argument checks and workspace sizes, through
the C ABI with addresses that are never read (every check comes before the
first CUDA call), and empty calls."""
import ctypes

import pytest

P = 1 << 20
BF16 = 1


def err(esa, rc, code, frag):
    assert rc == code, rc
    assert frag in esa._lib.load().esa_last_error().decode()


@pytest.mark.parametrize("kw,code,frag", [
    (dict(dtype=5), -1, "dtype"), (dict(id_bytes=2), -1, "id_bytes"), (dict(n=-1), -1, "shape"),
    (dict(vocab=0), -1, "vocab"), (dict(vocab=1 << 27), -2, "2^27"), (dict(n=1 << 31), -2, "2^30"),
    (dict(dim=12), -1, "16 bytes"), (dict(ids=None), -1, "ids"), (dict(ids=P + 4), -1, "ids"),
    (dict(scale=float("inf")), -1, "scale"), (dict(table=None), -1, "null"),
    (dict(table=P + 8), -1, "misaligned"), (dict(out=None), -1, "null")])
def test_embedding_refusals(esa, kw, code, frag):
    a = dict(dtype=BF16, id_bytes=8, n=2000, vocab=100, dim=64, ids=P, table=P, scale=1.0, out=P)
    a.update(kw)
    lib = esa._lib.load()
    rc = lib.esa_embedding_forward(a["dtype"], a["id_bytes"], a["n"], a["vocab"], a["dim"],
                                   a["ids"], a["table"], a["scale"], a["out"], None)
    err(esa, rc, code, frag)
    rc = lib.esa_embedding_backward(a["dtype"], a["id_bytes"], a["n"], a["vocab"], a["dim"],
                                    a["ids"], a["table"], a["scale"], -1, a["out"], P, 1 << 40,
                                    None)
    err(esa, rc, code, frag)


def test_embedding_workspace(esa):
    lib = esa._lib.load()
    size = lib.esa_embedding_backward_workspace_size
    assert size(0, 100, 64) == 0 and size(5, 100, 64) == 0
    n, V, d = 100000, 32000, 4096
    need = size(n, V, d)
    pieces = -(-n // 64)
    # keys and rows twice, head and tail partials of every piece, small tables
    assert 16 * n + 8 * pieces * d <= need <= 16 * n + 8 * pieces * d + (2 << 20)
    rc = lib.esa_embedding_backward(BF16, 8, n, V, d, P, P, 1.0, -1, P, P, need - 1, None)
    err(esa, rc, -4, "workspace")
    rc = lib.esa_embedding_backward(BF16, 8, n, V, d, P, P, 1.0, -1, P, None, need, None)
    err(esa, rc, -4, "workspace")
    rc = lib.esa_embedding_backward(BF16, 8, n, V, d, P, P, 1.0, -1, P, P + 16, need, None)
    err(esa, rc, -1, "256-byte")


def qk(esa, backward, **kw):
    lib = esa._lib.load()
    T = esa._lib.EsaTensor
    t = T(P, 4096, 64, 256)
    a = dict(dtype=BF16, B=2, L=16, D=64, q=t, Hq=4, k=t, Hk=2, wq=P, wk=P, eps=1e-6, pos=None, sb=0,
             inv=P, qo=t, ko=t, dwq=P, dwk=P, ws=P, wsb=1 << 30)
    a.update(kw)
    head = (a["dtype"], a["B"], a["L"], a["D"], a["q"], a["Hq"], a["k"], a["Hk"], a["wq"], a["wk"],
            a["eps"], a["pos"], a["sb"], a["inv"])
    if not backward:
        return lib.esa_qk_norm_rope_forward(*head, a["qo"], a["ko"], None)
    return lib.esa_qk_norm_rope_backward(*head, t, t, a["qo"], a["ko"], a["dwq"], a["dwk"], a["ws"],
                                         a["wsb"], None)


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("kw,code,frag", [
    (dict(dtype=9), -1, "dtype"), (dict(B=-1), -1, "negative"), (dict(sb=-1), -1, "negative"),
    (dict(D=48), -2, "head_dim"), (dict(D=8), -2, "head_dim"), (dict(D=512), -2, "head_dim"),
    (dict(dtype=0, D=256), -2, "head_dim"), (dict(eps=float("nan")), -1, "eps"),
    (dict(eps=-1e-6), -1, "eps"), (dict(inv=None), -1, "inv_freq"), (dict(wq=None), -1, "weight"),
    (dict(wk=P + 2), -1, "weight"), (dict(L=1 << 40), -2, "too many")])
def test_qk_refusals(esa, backward, kw, code, frag):
    err(esa, qk(esa, backward, **kw), code, frag)


@pytest.mark.parametrize("backward", [False, True])
def test_qk_refuses_misaligned_tensors(esa, backward):
    T = esa._lib.EsaTensor
    for name in ("q", "k", "qo", "ko"):
        err(esa, qk(esa, backward, **{name: T(P + 8, 4096, 64, 256)}), -1, "aligned")
        err(esa, qk(esa, backward, **{name: T(P, 4096, 60, 256)}), -1, "strides")
        err(esa, qk(esa, backward, **{name: T(None, 4096, 64, 256)}), -1, "null")


def test_qk_workspace_and_empty_calls(esa):
    lib = esa._lib.load()
    size = lib.esa_qk_norm_rope_backward_workspace_size
    assert size(0, 16, 4, 2, 64) == 0
    assert 0 < size(1, 1, 1, 0, 64) <= size(2, 16, 4, 2, 64) <= size(1, 1 << 20, 32, 8, 64) <= 1 << 20
    err(esa, qk(esa, True, wsb=16), -4, "workspace")
    err(esa, qk(esa, True, dwq=None), -1, "weight gradient")
    assert qk(esa, False, L=0) == 0 and qk(esa, False, Hq=0, Hk=0) == 0


@pytest.mark.parametrize("name", ["quantize", "dequantize", "norm_pack", "norm_unpack",
                                  "swiglu_pack", "swiglu_unpack"])
def test_pack_refusals(esa, name):
    lib = esa._lib.load()

    def call(dtype=BF16, fmt=0, n=4, dim=64, ptrs=None):
        p = dict(enumerate([P] * 8))
        p.update(ptrs or {})
        if name == "quantize":
            return lib.esa_quantize_rows(dtype, fmt, n, dim, p[0], p[1], p[2], None)
        if name == "dequantize":
            return lib.esa_dequantize_rows(dtype, fmt, n, dim, p[0], p[1], p[2], None)
        if name == "norm_pack":
            return lib.esa_rmsnorm_pack_forward(dtype, fmt, n, dim, p[0], p[3], p[4], p[1], 1e-6,
                                                p[2], p[5], p[6], p[7], None)
        if name == "norm_unpack":
            return lib.esa_rmsnorm_unpack_forward(dtype, fmt, n, dim, p[0], p[1], p[2], 1e-6, p[3],
                                                  p[4], p[5], None)
        if name == "swiglu_pack":
            return lib.esa_swiglu_pack_forward(dtype, fmt, n, dim, p[0], p[1], p[2], p[3], None)
        return lib.esa_swiglu_unpack_backward(dtype, fmt, n, dim, p[0], p[1], p[2], p[3], p[4],
                                              None)

    err(esa, call(dtype=3), -1, "dtype")
    err(esa, call(fmt=2), -1, "format")
    err(esa, call(n=-1), -1, "shape")
    err(esa, call(dim=4), -1, "16 bytes")
    for i in range(3):
        err(esa, call(ptrs={i: None}), -1, "null")
        err(esa, call(ptrs={i: P + 8}), -1, "misaligned")
    if name.startswith("norm"):
        err(esa, call(dim=16384), -2, "too large")
    assert call(n=0, ptrs={i: None for i in range(8)}) == 0


def test_python_refusals_before_the_device(esa):
    """Checks that need no device."""
    import torch
    ops = esa.layer_ops
    with pytest.raises(ValueError, match="int4"):
        ops.quantize_rows(torch.zeros(2, 8), "int4")
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.quantize_rows(torch.zeros(2, 8))
    p = ops.PackedRows(torch.zeros(2, 8, dtype=torch.uint8), torch.zeros(2, 2), "int8",
                       torch.float32)
    with pytest.raises(ValueError, match="scales"):
        ops.dequantize_rows(p)
    assert ctypes.sizeof(esa._lib.EsaTensor) == 32
