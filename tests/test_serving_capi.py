"""CPU: argument checks of the log probability, 4-bit weight and 4-bit cache entry
points, through the C ABI with addresses that are never read (every check comes
before the first CUDA call), and of their Python callers."""
import ctypes

import pytest
import torch

P = 1 << 20
BF16 = 1


def err(esa, rc, code, frag):
    assert rc == code, rc
    assert frag in esa._lib.load().esa_last_error().decode()


SCORE = dict(dtype=BF16, id_bytes=8, n=4, vocab=100, stride=100, logits=P, tokens=P, top=5, lp=P,
             ent=P, stats=P, ids=P, tlp=P)


def forward(esa, **kw):
    a = dict(SCORE, **kw)
    return esa._lib.load().esa_token_logprobs_forward(
        a["dtype"], a["id_bytes"], a["n"], a["vocab"], a["stride"], a["logits"], a["tokens"],
        a["top"], a["lp"], a["ent"], a["stats"], a["ids"], a["tlp"], None)


def backward(esa, **kw):
    a = dict(SCORE, dstride=100, out=P, **kw)
    return esa._lib.load().esa_token_logprobs_backward(
        a["dtype"], a["id_bytes"], a["n"], a["vocab"], a["stride"], a["logits"], a["tokens"],
        a["stats"], a["ent"], None, None, a["dstride"], a["out"], None)


@pytest.mark.parametrize("call", [forward, backward])
@pytest.mark.parametrize("kw,code,frag", [
    (dict(dtype=3), -1, "dtype"), (dict(id_bytes=2), -1, "id_bytes"), (dict(n=-1), -1, "shape"),
    (dict(vocab=0), -1, "shape"), (dict(stride=99), -1, "row stride"),
    (dict(vocab=1 << 31, stride=1 << 31), -2, "2^31"), (dict(n=1 << 29), -2, "2^28"),
    (dict(logits=None), -1, "logits"), (dict(logits=P + 1), -1, "logits"),
    (dict(tokens=None), -1, "tokens"), (dict(tokens=P + 4), -1, "tokens"),
    (dict(stats=None), -1, "null"), (dict(stats=P + 4), -1, "misaligned"),
    (dict(ent=None), -1, "null")])
def test_score_refusals(esa, call, kw, code, frag):
    err(esa, call(esa, **kw), code, frag)


@pytest.mark.parametrize("kw,frag", [
    (dict(top=33), "top_k"), (dict(top=-1), "top_k"), (dict(vocab=3, stride=3, top=4), "top_k"),
    (dict(lp=None), "output"), (dict(ids=None), "output"), (dict(tlp=None), "output")])
def test_score_forward_refusals(esa, kw, frag):
    err(esa, forward(esa, **kw), -1, frag)


def test_score_backward_refusals_and_empty_calls(esa):
    err(esa, backward(esa, dtype=0, logits=P + 2), -1, "logits")
    lib = esa._lib.load()

    def call(dstride, out, logits=P, n=4):
        return lib.esa_token_logprobs_backward(BF16, 8, n, 100, 128, logits, P, P, P, None, None,
                                               dstride, out, None)
    err(esa, call(99, P + 64), -1, "gradient row stride")
    err(esa, call(100, None), -1, "null")
    err(esa, call(100, P), -1, "in place")          # with another row stride
    assert call(100, None, n=0) == 0 and forward(esa, n=0, lp=None) == 0


W4 = dict(dtype=BF16, m=3, n=20, k=64, group=32, x=P, codes=P, scales=P, y=P)


@pytest.mark.parametrize("name", ["quantize", "dequantize", "linear"])
@pytest.mark.parametrize("kw,code,frag", [
    (dict(dtype=7), -1, "dtype"), (dict(n=0), -1, "shape"), (dict(k=0), -1, "shape"),
    (dict(k=12), -1, "16 bytes"), (dict(dtype=0, k=6), -1, "16 bytes"),
    (dict(n=(1 << 20) + 1), -2, "2^20"), (dict(k=1 << 21), -2, "2^20"), (dict(group=16), -1, "group"),
    (dict(codes=None), -1, "codes"), (dict(scales=P + 8), -1, "scales"), (dict(x=None), -1, "null"),
    (dict(x=P + 8), -1, "misaligned")])
def test_weight4_refusals(esa, name, kw, code, frag):
    a = dict(W4, **kw)
    lib = esa._lib.load()
    if name == "quantize":
        rc = lib.esa_quantize_weight4(a["dtype"], a["n"], a["k"], a["group"], a["x"], a["codes"],
                                      a["scales"], None)
    elif name == "dequantize":
        rc = lib.esa_dequantize_weight4(a["dtype"], a["n"], a["k"], a["group"], a["codes"],
                                        a["scales"], a["x"], None)
    else:
        rc = lib.esa_linear4(a["dtype"], a["m"], a["n"], a["k"], a["group"], a["x"], a["codes"],
                             a["scales"], a["y"], None)
    err(esa, rc, code, frag)


def test_weight4_sizes_and_rows(esa):
    lib = esa._lib.load()
    assert lib.esa_weight4_codes_size(0, 5) == 0
    assert lib.esa_weight4_codes_size(1, 8) == 1024
    assert lib.esa_weight4_codes_size(17, 136) == 4 * 1024
    call = lambda m, y=P: lib.esa_linear4(BF16, m, 20, 64, 32, P, P, P, y, None)
    err(esa, call(-1), -1, "n_rows")
    err(esa, call(1 << 21), -1, "n_rows")
    err(esa, call(2, None), -1, "null")
    assert call(0) == 0


def cache4(esa, name, **kw):
    lib = esa._lib.load()
    T = esa._lib.EsaTensor
    t = T(P, 4096, 64, 256)
    a = dict(dtype=BF16, codes=P, scales=P, B=2, Hkv=2, D=64, S=100, L=4, k=t, v=t, start=None,
             start0=0, counts=None, Hq=4, w=16, layer=1, layers=4, heads=0, offset=0, scale=0.1, q=t,
             o=t, lse=P, null=False)
    a.update(kw)
    c = esa._lib.EsaCache4(a["codes"], a["scales"], a["B"], a["Hkv"], a["D"], 0, a["S"])
    c = None if a["null"] else ctypes.byref(c)
    if name == "write":
        return lib.esa_cache4_write(a["dtype"], c, a["L"], a["k"], a["v"], a["start"], a["start0"],
                                    a["counts"], None)
    if name == "read":
        return lib.esa_cache4_read(a["dtype"], c, a["L"], a["k"], a["v"], a["start"], a["start0"],
                                   None)
    return lib.esa_cache4_forward(a["dtype"], c, a["Hq"], a["L"], a["w"], a["layer"], a["layers"],
                                  a["heads"], a["offset"], a["scale"], a["q"], a["start"],
                                  a["start0"], a["counts"], a["o"], a["lse"], None)


@pytest.mark.parametrize("name", ["write", "read", "forward"])
@pytest.mark.parametrize("kw,code,frag", [
    (dict(dtype=4), -1, "dtype"), (dict(null=True), -1, "null cache"), (dict(B=-1), -1, "shape"),
    (dict(Hkv=0), -1, "shape"), (dict(S=0), -1, "shape"), (dict(L=-1), -1, "shape"),
    (dict(D=32), -2, "head_dim"), (dict(D=96), -2, "head_dim"), (dict(S=(1 << 24) + 1), -2, "2^24"),
    (dict(L=(1 << 24) + 1), -1, "positions"), (dict(start0=-1), -1, "negative"),
    (dict(start=P + 4), -1, "start"), (dict(codes=None), -1, "codes"),
    (dict(scales=P + 2), -1, "scales")])
def test_cache_refusals(esa, name, kw, code, frag):
    err(esa, cache4(esa, name, **kw), code, frag)


@pytest.mark.parametrize("kw,code,frag", [
    (dict(Hq=3), -1, "divisible"), (dict(Hq=0), -1, "divisible"), (dict(w=0), -2, "attention_length"),
    (dict(w=2049), -2, "attention_length"), (dict(layers=0), -1, "layer"), (dict(layer=4), -1, "layer"),
    (dict(layer=-1), -1, "layer"), (dict(heads=3), -1, "pattern_heads"),
    (dict(offset=-1), -1, "head_offset"), (dict(heads=6, offset=3), -1, "pattern_heads"),
    (dict(scale=float("inf")), -1, "scale"), (dict(counts=P + 2), -1, "counts"),
    (dict(lse=None), -1, "lse")])
def test_cache_forward_refusals(esa, kw, code, frag):
    err(esa, cache4(esa, "forward", **kw), code, frag)


def test_cache_refuses_misaligned_tensors_and_takes_empty_calls(esa):
    T = esa._lib.EsaTensor
    for name, keys in (("write", "kv"), ("read", "kv"), ("forward", "qo")):
        for key in keys:
            err(esa, cache4(esa, name, **{key: T(P + 8, 4096, 64, 256)}), -1, "aligned")
            err(esa, cache4(esa, name, **{key: T(P, 4096, 60, 256)}), -1, "strides")
            err(esa, cache4(esa, name, **{key: T(None, 4096, 64, 256)}), -1, "null")
        assert cache4(esa, name, L=0) == 0 and cache4(esa, name, B=0) == 0
        err(esa, cache4(esa, name, B=70000), -2, "65535")


def test_python_callers_refuse_host_tensors_and_bad_shapes(esa):
    lops = esa.layer_ops
    with pytest.raises(RuntimeError, match="CUDA"):
        lops.token_logprobs(torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="CUDA"):
        lops.quantize_weight4(torch.zeros(8, 8))
    for bad in (dict(head_dim=32), dict(batch=-1), dict(max_len=0), dict(max_len=1 << 25),
                dict(num_kv_heads=0)):
        args = dict(dict(batch=1, num_kv_heads=1, max_len=8, head_dim=64), **bad)
        with pytest.raises(ValueError):
            esa.PackedKVCache(**args, device="cpu")
    cache = esa.PackedKVCache(2, 3, 10, 128, device="cpu")
    assert cache.nbytes() == 2 * 3 * 10 * 144
    with pytest.raises(RuntimeError, match="CUDA"):
        cache.write(torch.zeros(2, 3, 1, 128), torch.zeros(2, 3, 1, 128), 0)
    with pytest.raises(RuntimeError, match="CUDA"):
        esa.ops.forward_packed(torch.zeros(2, 3, 1, 128), cache, esa.PatternSpec(0, 1, 4), 1.0, 0)


@pytest.mark.parametrize("dtype,rows,way", [
    (torch.bfloat16, 64, "codes"), (torch.bfloat16, 65, "decoded"), (torch.float32, 65, "codes"),
    (torch.float32, 1 << 20, "codes"), (torch.float32, (1 << 20) + 1, "decoded")])
def test_how_the_packed_decoder_multiplies(esa, monkeypatch, dtype, rows, way):
    """The way that was measured to be faster, where the product takes so many rows."""
    taken = []
    monkeypatch.setattr(esa.layer_ops, "linear4", lambda x, w: taken.append("codes"))
    monkeypatch.setattr(esa.layer_ops, "dequantize_weight4",
                        lambda w, d: taken.append("decoded") or torch.zeros(1, 8, dtype=d))
    esa.PackedDecoder._project(torch.zeros(1, 8, dtype=dtype).expand(rows, 8), None)
    assert taken == [way]


@pytest.mark.parametrize("start", [-1, 1 << 63, 1 << 64, (1 << 64) + 3])
def test_a_start_beyond_64_bits_is_refused(esa, start):
    """It must not come out as another position."""
    with pytest.raises(ValueError, match="start"):
        esa.ops._span_args(2, start, None, torch.device("cpu"))
    assert esa.ops._span_args(2, (1 << 63) - 1, None, torch.device("cpu"))[1] == (1 << 63) - 1
