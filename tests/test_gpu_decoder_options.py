"""GPU: the decoder stack's options (scaled embedding with padding, query / key
norm, activations kept in 8 bits) against plain-torch restatements, and the
layer operators in the order a model uses them, decode included.

Tolerances as for the stack without options: float32 within 1e-4 (loss) and
1e-3 of each gradient's largest entry; the kernels' float32 sums differ from
torch's in their order only.
"""
import pytest
import torch
import torch.nn.functional as F

from decoder_reference import rmsnorm, rope, swiglu
from oracle import naive, pattern

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
CFG = dict(V=512, d=256, nl=3, Hq=4, Hkv=2, F=384, w=16, L=300, B=2, chunk=128)
EPS = 1e-6


class Stored:
    """The values of the 8-bit rows that a stack stored, in order.  The
    reference takes them from here instead of rounding its own activations:
    those differ from the stack's by float32 roundings, and where such a
    difference lies across the border between two codes the two would store
    values a whole step apart.  Each is checked against the reference's
    activation: within half a step of the format (int8: 1/254 of the group's
    largest; e4m3: 2^-4 of the value, or 2^-10 of a scale that is at most
    largest / 224) and the 1e-4 that the losses may differ by."""

    def __init__(self, monkeypatch, fmt):
        import elastic_sparse_attention_b200 as esa
        self.fmt, self.values = fmt, []
        lops = esa.layer_ops
        for name in ("rmsnorm_forward_packed", "swiglu_forward_packed"):
            def keep(*args, _f=getattr(lops, name), **kw):
                out = _f(*args, **kw)
                self.values.append(lops.dequantize_rows(out[-1], torch.float32))
                return out
            monkeypatch.setattr(lops, name, keep)

    def next(self, x):
        value = self.values.pop(0).view(x.shape)
        d = x.shape[-1]
        top = F.pad(x.abs(), (0, -d % 128)).unflatten(-1, (-1, 128)).amax(-1)
        top = top.repeat_interleave(128, -1)[..., :d]
        half = top / 254 if self.fmt == "int8" else torch.maximum(x.abs() * 2.0 ** -4,
                                                                  top / 224 * 2.0 ** -10)
        assert ((value - x).abs() <= half + 1e-4 * top).all()
        return value


def at(value, x):
    """x in the graph, ``value`` in the arithmetic."""
    return x + (value - x).detach()


def forward_of(exact, differentiated):
    """exact in the forward pass, the other's derivative in the backward."""
    return differentiated + (exact - differentiated).detach()


def attention_block(p, pre, y, i, cfg):
    B, L, _ = y.shape
    Hq, Hkv, D = cfg["Hq"], cfg["Hkv"], cfg["D"]
    positions = torch.arange(L, device=y.device)
    qkv = (y @ p[pre + "qkv_proj"].t()).view(B, L, Hq + 2 * Hkv, D)
    q, k = qkv[:, :, :Hq].transpose(1, 2), qkv[:, :, Hq:Hq + Hkv].transpose(1, 2)
    if pre + "q_norm" in p:
        q, k = rmsnorm(q, p[pre + "q_norm"], EPS), rmsnorm(k, p[pre + "k_norm"], EPS)
    q, k = rope(q, positions, cfg["inv_freq"]), rope(k, positions, cfg["inv_freq"])
    v = qkv[:, :, Hq + Hkv:].transpose(1, 2)
    idx, mask, _ = pattern.prepared_indices(Hq, cfg["w"], i, cfg["nl"], L, L, L)
    o, _ = naive.naive_forward(q, k, v, torch.from_numpy(idx).to(y.device),
                               torch.from_numpy(mask).to(y.device), D ** -0.5, Hq // Hkv)
    return o.transpose(1, 2).reshape(B, L, Hq * D) @ p[pre + "o_proj"].t()


def mlp(p, pre, y, stored):
    gu = y @ p[pre + "gate_up_proj"].t()
    down = p[pre + "down_proj"].t()
    if stored is None:
        return swiglu(gu) @ down
    value = stored.next(gu.detach().unflatten(-1, (2, -1))).flatten(-2)
    return forward_of(swiglu(gu) @ down, swiglu(at(value, gu)) @ down)


def layer(p, i, h, y, cfg, mlp_stored):
    pre = f"layers.{i}."
    h = h + attention_block(p, pre, y, i, cfg)
    y = rmsnorm(h, p[pre + "post_attention_norm"], EPS)
    h = h + mlp(p, pre, y, mlp_stored)
    w = p[f"layers.{i + 1}.input_norm"] if i + 1 < cfg["nl"] else p["final_norm"]
    return h, rmsnorm(h, w, EPS)


def reference_loss(p, ids, labels, cfg, scale=1.0, pad=None, stored=None, ckpt=False):
    h = F.embedding(ids, p["embed"], padding_idx=pad) * scale
    w0 = p["layers.0.input_norm"]
    y = rmsnorm(h, w0, EPS)
    for i in range(cfg["nl"]):
        exact = layer(p, i, h, y, cfg, None if ckpt else stored)
        if stored and ckpt:
            hd = stored.next(h.detach())
            if i == 0:
                y = forward_of(y, rmsnorm(at(hd, h), w0, EPS))
            yd = rmsnorm(hd, p[f"layers.{i}.input_norm"].detach(), EPS)
            again = layer(p, i, at(hd, h), at(yd, y), cfg, None)
            h, y = (forward_of(a, b) for a, b in zip(exact, again))
        else:
            h, y = exact
    logits = y @ p["lm_head"].t()
    return F.cross_entropy(logits[:, :-1].reshape(-1, logits.shape[-1]), labels[:, 1:].reshape(-1))


def build(dtype=torch.float32, cfg=CFG, **kw):
    import elastic_sparse_attention_b200 as esa
    m = esa.ElasticDecoderStack(vocab_size=cfg["V"], hidden_size=cfg["d"],
                                num_hidden_layers=cfg["nl"], num_attention_heads=cfg["Hq"],
                                num_key_value_heads=cfg["Hkv"], intermediate_size=cfg["F"],
                                attention_length=cfg["w"], max_seq_len=cfg["L"],
                                loss_chunk_rows=cfg["chunk"], dtype=dtype, device=DEV, seed=3, **kw)
    if kw.get("qk_norm"):
        g = torch.Generator().manual_seed(8)
        with torch.no_grad():
            for lw in m.layers:
                for w in (lw.q_norm, lw.k_norm):
                    w.copy_(1 + 0.3 * torch.randn(w.shape, generator=g))
    g = torch.Generator().manual_seed(7)
    ids = torch.randint(1, cfg["V"], (cfg["B"], cfg["L"]), generator=g).to(DEV)
    return m, ids


OPTIONS = [
    dict(embed_scale=16.0), dict(embed_scale=2.5, padding_idx=0), dict(padding_idx=3),
    dict(qk_norm=True), dict(qk_norm=True, embed_scale=16.0, activation_checkpointing=True),
    dict(activation_storage="int8"), dict(activation_storage="e4m3", qk_norm=True),
    dict(activation_storage="int8", activation_checkpointing=True),
    dict(activation_storage="e4m3", activation_checkpointing=True, qk_norm=True, embed_scale=16.0,
         padding_idx=0),
]


@pytest.mark.parametrize("kw", OPTIONS, ids=lambda kw: "-".join(f"{k}={v}" for k, v in kw.items()))
def test_stack_options_match_reference(kw, monkeypatch):
    m, ids = build(**kw)
    fmt = kw.get("activation_storage")
    stored = Stored(monkeypatch, fmt) if fmt else None
    pad = kw.get("padding_idx")
    if pad is not None:
        ids[:, -40:] = pad
    loss = m(ids, labels=ids)
    if stored:                                 # what the forward pass stored
        monkeypatch.undo()
    loss.backward()
    p = {n: t.detach().clone().requires_grad_(True) for n, t in m.named_parameters()}
    cfg = dict(CFG, D=CFG["d"] // CFG["Hq"], inv_freq=m.inv_freq)
    ref = reference_loss(p, ids, ids, cfg, scale=kw.get("embed_scale", 1.0), pad=pad,
                         stored=stored, ckpt=kw.get("activation_checkpointing"))
    ref.backward()
    assert not stored or not stored.values
    assert abs(loss.item() - ref.item()) <= 1e-4 * abs(ref.item())
    for n, t in m.named_parameters():
        want = p[n].grad
        err = (t.grad - want).abs().max().item()
        assert err <= 1e-3 * want.abs().max().item() + 1e-7, f"{n}: {err:.3e}"
    if pad is not None:
        assert not m.embed.grad[pad].any()


def test_8_bit_storage_leaves_the_forward_pass_alone():
    m, ids = build()
    want = m(ids, labels=ids)
    hidden = m(ids)
    for ckpt in (False, True):
        for fmt in ("int8", "e4m3"):
            n, _ = build(activation_storage=fmt, activation_checkpointing=ckpt)
            assert torch.equal(n(ids, labels=ids), want)
            with torch.no_grad():
                assert torch.equal(n(ids), hidden)


def test_8_bit_storage_keeps_less_memory():
    """What a forward pass leaves for the backward: with 8-bit gate / up rows
    3 of the 4 bytes of a float32 element are saved; with 8-bit checkpoints a
    layer keeps one byte per element of its input instead of two rows."""
    def kept(**kw):
        m, ids = build(**kw)
        m(ids, labels=ids).backward()      # the key plans and workspaces settle
        # the bytes asked for: the allocator's own blocks may be up to 1 MiB larger
        held = lambda: torch.cuda.memory_stats()["requested_bytes.all.current"]
        before = held()
        loss = m(ids, labels=ids)
        return held() - before, loss

    rows = CFG["B"] * CFG["L"]
    plain, _ = kept()
    packed, _ = kept(activation_storage="int8")
    assert plain - packed >= CFG["nl"] * rows * 2 * CFG["F"] * 3 * 0.9
    ckpt, _ = kept(activation_checkpointing=True)
    ckpt8, _ = kept(activation_checkpointing=True, activation_storage="int8")
    assert ckpt - ckpt8 >= (CFG["nl"] - 1) * rows * CFG["d"] * 6


def test_bf16_training_step_with_every_option():
    """Runs at the module's width in bf16; gradients finite, present for every
    parameter, and near those of the stack that keeps everything."""
    cfg = dict(CFG, L=520, w=64, d=512, Hq=4, Hkv=4, F=1024, nl=4)
    grads = []
    for fmt in (None, "int8"):
        m, ids = build(torch.bfloat16, cfg, qk_norm=True, embed_scale=512 ** 0.5, padding_idx=0,
                       activation_checkpointing=True, activation_storage=fmt)
        m(ids, labels=ids).backward()
        assert all(p.grad is not None and p.grad.isfinite().all() for p in m.parameters())
        grads.append(torch.cat([p.grad.float().flatten() for p in m.parameters()]))
    assert F.cosine_similarity(grads[0], grads[1], dim=0).item() > 0.99


def test_frozen_parameters_with_8_bit_checkpoints():
    m, ids = build(activation_checkpointing=True, activation_storage="int8")
    m.layers[1].gate_up_proj.requires_grad_(False)
    m.layers[0].input_norm.requires_grad_(False)
    m(ids, labels=ids).backward()
    assert m.layers[1].gate_up_proj.grad is None and m.layers[0].input_norm.grad is None
    assert m.layers[1].down_proj.grad.abs().max() > 0 and m.embed.grad.abs().max() > 0


def test_overflow_stays_visible_with_8_bit_checkpoints():
    """An infinity in a layer's input makes gradients that a loss scaler sees."""
    m, ids = build(activation_checkpointing=True, activation_storage="int8")
    with torch.no_grad():
        m.embed[ids[0, 5], 3] = float("inf")
    m(ids, labels=ids).backward()
    assert not m.embed.grad.isfinite().all()


def test_options_are_checked():
    with pytest.raises(ValueError):
        build(activation_storage="int4")
    with pytest.raises(ValueError):
        build(padding_idx=512)


def test_decode_step_into_a_key_cache():
    """Prefill of a cache, then single tokens: embedding, query / key norm with
    the key written into its cache rows, attention over the cache; the same
    outputs as the whole sequence at once."""
    import elastic_sparse_attention_b200 as esa
    lops, dt = esa.layer_ops, torch.bfloat16
    B, L, Hq, Hkv, D, w, V = 2, 140, 4, 2, 64, 16, 300
    d = Hq * D
    g = torch.Generator().manual_seed(2)
    table, proj = (0.3 * torch.randn(n, d, generator=g).to(DEV, dt)
                   for n in (V, (Hq + 2 * Hkv) * D))
    wq, wk = ((1 + 0.2 * torch.randn(D, generator=g)).to(DEV, dt) for _ in range(2))
    inv = lops.rope_inv_freq(D, 10000.0, DEV)
    ids = torch.randint(0, V, (B, L), generator=g).to(DEV)
    attn = esa.ElasticSparseAttention(2, 4, Hq, D, w, L, num_key_value_heads=Hkv)

    def heads(tokens):
        x = lops.embedding_forward(tokens, table, d ** 0.5)
        qkv = (x @ proj.t()).view(B, tokens.shape[1], Hq + 2 * Hkv, D)
        return (qkv[:, :, :Hq].transpose(1, 2), qkv[:, :, Hq:Hq + Hkv].transpose(1, 2),
                qkv[:, :, Hq + Hkv:].transpose(1, 2))

    q, k, v = heads(ids)
    q2, k2 = lops.qk_norm_rope(q, k, wq, wk, EPS, inv)
    whole, _ = attn(q2, k2, v)
    kc = torch.zeros(B, Hkv, L, D, device=DEV, dtype=dt)
    vc = torch.zeros_like(kc)
    n = 137
    kc[:, :, :n], vc[:, :, :n] = k2[:, :, :n], v[:, :, :n]
    for t in range(n, L):
        q, k, v = heads(ids[:, t:t + 1])
        pos = torch.tensor([t], device=DEV)
        q1, _ = lops.qk_norm_rope(q, k, wq, wk, EPS, inv, positions=pos, k_out=kc[:, :, t:t + 1])
        vc[:, :, t:t + 1] = v
        out, _ = attn(q1, kc[:, :, :t + 1], vc[:, :, :t + 1], cache_position=pos)
        # two kernels of the same bf16 attention: a step of bf16 at the outputs' size (the
        # projections' sums may round differently for one row and for many)
        assert (out - whole[:, t:t + 1]).float().abs().max() <= 2.0 ** -6 * whole.abs().max()
    assert esa.ops.device_errors() == 0
