"""What is timed of the operators that answer and serve in few bits: log
probabilities of given tokens with entropy and top alternatives and their
gradient, products with weights of 4 bits, and a key / value cache of 4 bits
with the elastic attention that reads it.

``own`` chooses who computes: False runs elementary torch operations (the
plain form), True the framework's kernels.

Every case is a dict with ``kind`` (which operator and direction), ``dtype``
and the sizes of its kind:

  score, score_grad     rows x V logits, one token each; top (alternatives per
                        row), masked (share of the vocabulary at -inf),
                        ignored (share of rows whose token is -100)
  linear4               M rows x K times a weight [N, K] in 4 bits, a scale per
                        ``group`` elements
  cache_write           L rows written per sequence and read back; B sequences,
                        Hkv heads of D, S cache rows
  cache_attend          L query rows per sequence with Hq heads, attention
                        length w, layer ``layer`` of ``layers``

``ragged``: the sequences of a batch bring different numbers of rows (the last
of three or more none), the rest of their L rows is padding.

4 bits: each group of consecutive elements of a row has the scale s = the
bfloat16 nearest to float32(max|x| / 7), at least 2^-126, and the codes n = the
integer nearest to x / s, ties to even; a code stands for n * s.
"""
import functools
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
IGNORED = -100
CACHE_GROUP = 32     # elements of a cached head row that share a scale
TINY = 2.0 ** -126


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one decode step of a batch of 8: the sampled tokens' log probabilities
        # with 20 alternatives for the answer
        dict(name="score_decode", kind="score", dtype="bf16", rows=8, V=32000, top=20, masked=0.0,
             ignored=0.0),
        # answers constrained to a part of an odd vocabulary, float32 logits
        dict(name="score_masked", kind="score", dtype="fp32", rows=333, V=50021, top=8, masked=0.3,
             ignored=0.0),
        # scoring a long text: one chunk of the stack's LM head
        dict(name="score_prompt", kind="score", dtype="bf16", rows=8192, V=32000, top=5,
             masked=0.0, ignored=0.1),
        # policy gradient with an entropy term in a small fp32 model
        dict(name="score_grad_small", kind="score_grad", dtype="fp32", rows=300, V=512, top=0,
             masked=0.0, ignored=0.1),
        # the same for one chunk of the stack's LM head
        dict(name="score_grad_long", kind="score_grad", dtype="bf16", rows=8192, V=32000, top=0,
             masked=0.0, ignored=0.1),
        # one token through the stack's fused query / key / value projection
        dict(name="linear4_one", kind="linear4", dtype="bf16", M=1, K=4096, N=12288, group=128),
        # a few rows of a small fp32 model, odd sizes, ragged last group
        dict(name="linear4_odd", kind="linear4", dtype="fp32", M=5, K=1000, N=777, group=32),
        # a decode batch of 32 through the stack's MLP down projection
        dict(name="linear4_batch", kind="linear4", dtype="fp16", M=32, K=11008, N=4096, group=128),
        # one new token for each of 64 sequences
        dict(name="cache_write_decode", kind="cache_write", dtype="bf16", B=64, L=1, Hkv=8, D=128,
             S=4096, ragged=False),
        # three prompts of different lengths, padded to one
        dict(name="cache_write_prompt", kind="cache_write", dtype="fp16", B=3, L=20011, Hkv=8,
             D=128, S=20480, ragged=True),
        # one new token for each of 8 sequences deep in a long context
        dict(name="cache_attend_decode", kind="cache_attend", dtype="bf16", B=8, L=1, Hq=32, Hkv=8,
             D=128, S=131072, w=64, layer=4, layers=8, ragged=False),
        # a chunk of a long prompt against the cache of what came before
        dict(name="cache_attend_prompt", kind="cache_attend", dtype="bf16", B=1, L=4096, Hq=32,
             Hkv=8, D=128, S=131072, w=64, layer=4, layers=8, ragged=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["score", "score", "score_grad", "linear4", "linear4", "cache_write",
                       "cache_attend", "cache_attend"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    case = dict(kind=kind, dtype=dtype)
    if kind in ("score", "score_grad"):
        V = _log(rng, 100, 131072)
        rows = _log(rng, 1, min(16384, (1 << 28) // (V * BYTES[dtype] // 2)))
        case.update(rows=rows, V=V, top=rng.choice([0, 1, 5, 20, 32]) if kind == "score" else 0,
                    masked=rng.choice([0.0, 0.0, 0.3]), ignored=rng.choice([0.0, 0.1]))
    elif kind == "linear4":
        K = 8 * _log(rng, 4, 2048)
        N = _log(rng, 8, min(32768, (1 << 26) // K))
        case.update(M=_log(rng, 1, 64), K=K, N=N, group=rng.choice([32, 64, 128, 128]))
    elif kind == "cache_write":
        D = rng.choice([64, 128, 128, 256])
        B, Hkv = rng.choice([1, 2, 3, 8, 33]), rng.choice([1, 2, 8])
        L = _log(rng, 1, min(32768, (1 << 25) // (B * Hkv * D)))
        case.update(B=B, L=L, Hkv=Hkv, D=D, S=L + _log(rng, 1, 2048), ragged=rng.random() < 0.5)
    else:
        D = rng.choice([64, 128, 128, 256])
        Hkv = rng.choice([1, 2, 4, 8])
        Hq = Hkv * rng.choice([1, 2, 4])
        w = rng.choice([16, 33, 64, 64, 100, 256])
        B = rng.choice([1, 1, 2, 3, 8])
        L = _log(rng, 1, min(4096, max(1, (1 << 29) // (B * Hq * w * D))))
        S = L + _log(rng, 64, min(131072, (1 << 27) // (B * Hkv * D)))
        layers = rng.choice([4, 8, 12])
        case.update(B=B, L=L, Hq=Hq, Hkv=Hkv, D=D, S=S, w=w, layer=rng.randrange(layers),
                    layers=layers, ragged=rng.random() < 0.5)
    return case


def _starts(case):
    """The first of the L rows of each sequence, the later sequences a little shorter."""
    return [max(0, case["S"] - case["L"] - 97 * b) for b in range(case["B"])]


def _counts(case):
    B, L = case["B"], case["L"]
    if not case["ragged"]:
        return [L] * B
    return [0 if b == B - 1 and B > 2 else L - L * b // (2 * B) for b in range(B)]


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _codes(x, group):
    """(codes, scales) of the plain form: int8 and float32, a scale per group."""
    pad = -x.shape[-1] % group
    xf = torch.nn.functional.pad(x.float(), (0, pad)).unflatten(-1, (-1, group))
    top = xf.abs().amax(-1, keepdim=True)
    # by a tensor: a division by a number may be a product with its inverse
    scale = (top / torch.full_like(top, 7.0)).to(torch.bfloat16).float().clamp_min(TINY)
    # quotients next to a border between two codes need 64 bits
    code = torch.round(xf.double() / scale.double()).to(torch.int8)
    return code.flatten(-2)[..., :x.shape[-1]].contiguous(), scale[..., 0].contiguous()


def _values(codes, scales, group):
    return codes.float() * scales.repeat_interleave(group, -1)[..., :codes.shape[-1]]


def _head_rows(shape, g, dev, dt):
    """Gaussian head rows with a few large channels, one sequence at a time."""
    out = torch.empty(shape, dtype=dt, device=dev)
    gain = torch.where(torch.rand(shape[1], 1, shape[-1], generator=g, device=dev) < 0.03, 6.0, 1.0)
    for b in range(shape[0]):
        out[b] = torch.randn(shape[1:], generator=g, device=dev) * gain
    return out


def _logits(case, g, dev, dt):
    """Logits as a language model gives them: spread by about 2.5, the given token
    mostly among the likely ones."""
    rows, V = case["rows"], case["V"]
    x = torch.empty(rows, V, dtype=dt, device=dev)
    tokens = torch.randint(0, V, (rows,), generator=g, device=dev)
    for r in range(0, rows, 1024):
        z = 2.5 * torch.randn(min(1024, rows - r), V, generator=g, device=dev)
        t = tokens[r:r + 1024, None]
        if case["masked"]:
            z.masked_fill_(torch.rand(z.shape, generator=g, device=dev) < case["masked"],
                           -math.inf)
        z.scatter_(1, t, 6 + 3 * torch.randn(t.shape, generator=g, device=dev))
        x[r:r + 1024] = z
    if case["ignored"]:
        tokens[torch.rand(rows, generator=g, device=dev) < case["ignored"]] = IGNORED
    return x, tokens


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    s = dict(case=case)
    kind = case["kind"]
    if kind in ("score", "score_grad"):
        s["logits"], s["tokens"] = _logits(case, g, dev, dt)
        if kind == "score_grad":
            s["dlogprobs"] = torch.randn(case["rows"], generator=g, device=dev)
            s["dentropy"] = 0.01 * torch.randn(case["rows"], generator=g, device=dev)
    elif kind == "linear4":
        w = (0.02 * torch.randn(case["N"], case["K"], generator=g, device=dev)).to(dt)
        s["x"] = torch.randn(case["M"], case["K"], generator=g, device=dev).to(dt)
        if own:
            from elastic_sparse_attention_b200 import layer_ops
            s["weight"] = layer_ops.quantize_weight4(w, group=case["group"])
        else:
            s["codes"], s["scales"] = _codes(w, case["group"])
    else:
        B, L, Hkv, D, S = (case[n] for n in ("B", "L", "Hkv", "D", "S"))
        starts, counts = _starts(case), _counts(case)
        s["start"] = torch.tensor(starts, device=dev)
        s["counts"] = torch.tensor(counts, device=dev) if case["ragged"] else None
        k = _head_rows((B, Hkv, S, D), g, dev, dt)       # what the cache holds before the call
        v = _head_rows((B, Hkv, S, D), g, dev, dt)
        if own:
            from elastic_sparse_attention_b200 import PackedKVCache
            s["cache"] = PackedKVCache(B, Hkv, S, D, device=dev)
            s["cache"].write(k, v, 0)
        else:
            s["cache"] = [_codes_by_sequence(t) for t in (k, v)]
        del k, v
        if kind == "cache_write":
            # rows of a fused projection: [B, L, heads, D] in memory
            kv = torch.randn(B, L, 2 * Hkv, D, generator=g, device=dev).to(dt)
            s["k"] = kv[:, :, :Hkv].transpose(1, 2)
            s["v"] = kv[:, :, Hkv:].transpose(1, 2)
        else:
            s["q"] = (2 * torch.randn(B, L, case["Hq"], D, generator=g, device=dev)
                      ).to(dt).transpose(1, 2)
    return s


def _codes_by_sequence(x):
    codes = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    scales = torch.empty(x.shape[:-1] + (x.shape[-1] // CACHE_GROUP,), device=x.device)
    step = max(1, (1 << 25) // (x.shape[1] * x.shape[-1]))
    for b in range(x.shape[0]):
        for r in range(0, x.shape[2], step):
            codes[b, :, r:r + step], scales[b, :, r:r + step] = _codes(x[b, :, r:r + step],
                                                                       CACHE_GROUP)
    return codes, scales


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------
def _run_own(s):
    from elastic_sparse_attention_b200 import PatternSpec, layer_ops, ops
    case = s["case"]
    kind = case["kind"]
    if kind == "score":
        r = layer_ops.token_logprobs(s["logits"], s["tokens"], top_k=case["top"])
        return (r.logprobs, r.entropy) + ((r.top_ids, r.top_logprobs) if case["top"] else ())
    if kind == "score_grad":
        r = layer_ops.token_logprobs(s["logits"], s["tokens"])
        return r.logprobs, r.entropy, layer_ops.token_logprobs_backward(
            s["logits"], s["tokens"], r, s["dlogprobs"], s["dentropy"])
    if kind == "linear4":
        return layer_ops.linear4(s["x"], s["weight"])
    if kind == "cache_write":
        s["cache"].write(s["k"], s["v"], s["start"], s["counts"])
        return s["cache"].read(s["start"], case["L"], DTYPES[case["dtype"]])
    spec = PatternSpec(case["layer"], case["layers"], case["w"])
    return ops.forward_packed(s["q"], s["cache"], spec, case["D"] ** -0.5, s["start"], s["counts"])


# ---------------------------------------------------------------------------
# the plain form
# ---------------------------------------------------------------------------
def _score_plain(x, tokens, top):
    z = x.float()
    m = z.amax(-1, keepdim=True)
    e = torch.exp(z - m)
    total = e.sum(-1, keepdim=True)
    lp = z - (m + torch.log(total))
    p = e / total
    entropy = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(-1)
    picked = lp.gather(1, tokens.clamp_min(0)[:, None])[:, 0]
    picked = torch.where(tokens == IGNORED, torch.zeros_like(picked), picked)
    out = [picked, entropy]
    if top:
        ids = torch.sort(z, dim=-1, descending=True, stable=True).indices[:, :top].clone()
        out += [ids, lp.gather(1, ids)]
    return out, lp, p


def _indices_plain(case, pos):
    """Key positions and mask [rows, Hq, w] of query positions [rows]: every step in
    float32, rounding half to even."""
    w, H = case["w"], case["Hq"]
    alpha = case["layer"] / max(case["layers"] - 1, 1)
    dev = pos.device
    f = functools.partial(torch.tensor, dtype=torch.float32, device=dev)
    edge = (pos.clamp_min(w - 1) + 1).float()
    span = f(w * (1 - alpha)) + edge * f(alpha)
    first = torch.round(edge - span).clamp_min(0)
    step = (edge - first) / f(float(w))
    slots = torch.arange(w + 1, device=dev).float()
    grid = first[:, None] + torch.round(slots * step[:, None])             # [rows, w + 1]
    t = (torch.arange(H, device=dev).float() / f(float(max(H - 1, 1))))[None, :, None]
    idx = torch.round(grid[:, None, :-1] * (1 - t) + (grid[:, None, 1:] - 1) * t).long()
    return idx, idx <= pos[:, None, None]


def _attend_plain(s):
    case = s["case"]
    B, L, Hq, Hkv, D = (case[n] for n in ("B", "L", "Hq", "Hkv", "D"))
    q = s["q"]
    o = torch.zeros(B, L, Hq, D, dtype=q.dtype, device=q.device)
    lse = torch.full((B, Hq, L), -math.inf, device=q.device)
    head = (torch.arange(Hq, device=q.device) // (Hq // Hkv))[None, :, None]
    step = max(1, (1 << 26) // (Hq * case["w"] * D))
    for b, (start, count) in enumerate(zip(_starts(case), _counts(case))):
        for r in range(0, count, step):
            n = min(step, count - r)
            idx, keep = _indices_plain(case, start + r + torch.arange(n, device=q.device))
            rows = torch.where(keep, idx, torch.zeros_like(idx))
            k, v = (_values(c[b][head, rows], f[b][head, rows], CACHE_GROUP)
                    for c, f in s["cache"])
            score = (q[b, :, r:r + n].transpose(0, 1).float()[:, :, None] * k).sum(-1)
            score = (score * D ** -0.5).masked_fill(~keep, -math.inf)
            m = score.amax(-1, keepdim=True)
            e = torch.exp(score - m)
            total = e.sum(-1, keepdim=True)
            o[b, r:r + n] = ((e / total)[..., None] * v).sum(-2).to(q.dtype)
            lse[b, :, r:r + n] = ((m + torch.log(total))[..., 0] / math.log(2)).t()
    return o.transpose(1, 2), lse


def _run_plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind in ("score", "score_grad"):
        parts, grads = [], []
        for r in range(0, case["rows"], 1024):
            x, t = s["logits"][r:r + 1024], s["tokens"][r:r + 1024]
            out, lp, p = _score_plain(x, t, case["top"])
            parts.append(out)
            if kind == "score_grad":
                valid = t != IGNORED
                g = torch.where(valid, s["dlogprobs"][r:r + 1024], 0.0)[:, None]
                h = s["dentropy"][r:r + 1024, None]
                safe = torch.where(p > 0, lp, torch.zeros_like(lp))
                d = -p * (g + h * (safe + out[1][:, None]))
                d.scatter_add_(1, t.clamp_min(0)[:, None], g)
                grads.append(d.to(x.dtype))
        out = tuple(torch.cat(p) for p in zip(*parts))
        return out + ((torch.cat(grads),) if grads else ())
    if kind == "linear4":
        w = _values(s["codes"], s["scales"], case["group"])
        return (s["x"].float() @ w.t()).to(s["x"].dtype)
    if kind == "cache_write":
        dev = s["start"].device
        at = s["start"][:, None] + torch.arange(case["L"], device=dev)            # [B, L]
        given = torch.arange(case["L"], device=dev) < torch.tensor(_counts(case), device=dev)[:, None]
        given = given[..., None, None]
        seq = torch.arange(case["B"], device=dev)[:, None]
        outs = []
        for x, (codes, scales) in zip((s["k"], s["v"]), s["cache"]):
            c, f = _codes(x.transpose(1, 2), CACHE_GROUP)                          # [B, L, Hkv, ...]
            c = torch.where(given, c, codes[seq, :, at])
            f = torch.where(given, f, scales[seq, :, at])
            codes[seq, :, at], scales[seq, :, at] = c, f
            outs.append(_values(c, f, CACHE_GROUP).to(x.dtype).transpose(1, 2))
        return tuple(outs)
    return _attend_plain(s)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def _pattern64(case, pos):
    """Key positions [rows, Hq, w] and mask of one or more query positions (numpy):
    the pattern is defined in float32 steps."""
    f32 = np.float32
    w, H = case["w"], case["Hq"]
    a = case["layer"] / max(case["layers"] - 1, 1)
    pos = np.asarray(pos, dtype=np.int64)
    last = np.maximum(pos, w - 1) + 1
    e = last.astype(f32)
    width = f32(w * (1 - a)) + e * f32(a)
    lo = np.maximum(np.rint(e - width), f32(0)).astype(np.int64)
    gap = (last - lo).astype(f32) / f32(w)
    at = lo[:, None] + np.rint(np.arange(w + 1).astype(f32)[None] * gap[:, None]).astype(np.int64)
    mix = np.arange(H).astype(f32) / f32(max(H - 1, 1))
    left = at[:, None, :-1].astype(f32) * (f32(1) - mix)[None, :, None]
    right = (at[:, None, 1:] - 1).astype(f32) * mix[None, :, None]
    idx = np.rint(left + right).astype(np.int64)
    return idx, idx <= pos[:, None, None]


@functools.lru_cache(maxsize=64)
def _cache_rows_read(items):
    """Distinct (sequence, key / value head, position) that a case's queries attend to."""
    case = dict(items)
    total = 0
    per = case["Hq"] // case["Hkv"]
    for start, count in zip(_starts(case), _counts(case)):
        seen = np.zeros((case["Hkv"], case["S"]), dtype=bool)
        for r in range(0, count, 512):
            idx, keep = _pattern64(case, start + np.arange(r, min(count, r + 512)))
            for h in range(case["Hq"]):
                seen[h // per, idx[:, h][keep[:, h]]] = True
        total += int(seen.sum())
    return total


def work(case):
    es = BYTES[case["dtype"]]
    kind = case["kind"]
    if kind in ("score", "score_grad"):
        n, rows = case["rows"] * case["V"], case["rows"]
        if kind == "score":
            return {"bytes": n * es + rows * (16 + 12 * case["top"]), "flops": 6 * n}
        return {"bytes": 2 * n * es + rows * 24, "flops": 13 * n}
    if kind == "linear4":
        M, K, N = case["M"], case["K"], case["N"]
        return {"bytes": N * (K // 2) + N * -(-K // case["group"]) * 2 + (M * K + M * N) * es,
                "flops": 2 * M * K * N}
    D, Hkv = case["D"], case["Hkv"]
    row = 2 * (D // 2 + D // CACHE_GROUP * 2)            # key and value, codes and scales
    if kind == "cache_write":
        written, read = sum(_counts(case)) * Hkv, case["B"] * case["L"] * Hkv
        return {"bytes": written * (2 * D * es + row) + read * (row + 2 * D * es),
                "flops": (written * 8 + read) * 2 * D}
    pairs = sum(_counts(case)) * case["Hq"]
    rows = _cache_rows_read(tuple(sorted(case.items())))
    return {"bytes": rows * row + case["B"] * case["L"] * case["Hq"] * (D * es + 4)
            + pairs * D * es, "flops": 4 * pairs * case["w"] * D}


# ---------------------------------------------------------------------------
# the definition, in 64 bits
# ---------------------------------------------------------------------------
def _decoded64(x, group):
    """Group by group: codes n = nearest integer (ties to even) of x / s, with s the
    bfloat16 nearest to the float32 quotient max|x| / 7."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for lo in range(0, x.shape[-1], group):
        v = x[..., lo:lo + group].double()
        top = v.abs().max(-1, keepdim=True).values
        s = torch.clamp((top / 7).float().bfloat16().double(), min=TINY)
        out[..., lo:lo + group] = torch.round(v / s) * s
    return out


def _attend64(case, s, k, v):
    """k, v: the rows the cache was filled with."""
    B, L, Hq, Hkv, D = (case[n] for n in ("B", "L", "Hq", "Hkv", "D"))
    q = s["q"].double()
    o = torch.zeros(B, Hq, L, D, dtype=torch.float64, device=q.device)
    lse = torch.full((B, Hq, L), -math.inf, dtype=torch.float64, device=q.device)
    per = Hq // Hkv
    step = max(1, (1 << 24) // (case["w"] * D))
    for b, (start, count) in enumerate(zip(_starts(case), _counts(case))):
        for r in range(0, count, step):
            n = min(step, count - r)
            idx, keep = _pattern64(case, start + np.arange(r, r + n))
            idx = torch.from_numpy(np.where(keep, idx, 0)).to(q.device)
            keep = torch.from_numpy(keep).to(q.device)
            for h in range(Hq):
                kk = _decoded64(k[b, h // per][idx[:, h]], CACHE_GROUP)
                vv = _decoded64(v[b, h // per][idx[:, h]], CACHE_GROUP)
                score = torch.einsum("rd,rwd->rw", q[b, h, r:r + n], kk) / math.sqrt(D)
                score[~keep[:, h]] = -math.inf
                o[b, h, r:r + n] = torch.einsum("rw,rwd->rd", torch.softmax(score, -1), vv)
                lse[b, h, r:r + n] = torch.logsumexp(score, -1) / math.log(2)
    return o, lse


def exact(case, seed):
    kind = case["kind"]
    dt = DTYPES[case["dtype"]]
    dev = torch.device("cuda")
    if kind in ("score", "score_grad"):
        s = prepare(case, seed)
        outs = []
        for r in range(0, case["rows"], 512):
            z = s["logits"][r:r + 512].double()
            t = s["tokens"][r:r + 512]
            given = t != IGNORED
            lp = torch.log_softmax(z, -1)
            p = lp.exp()
            ent = -(p * lp).nan_to_num(0.0).sum(-1)
            out = [lp[torch.arange(len(t), device=dev), t * given] * given, ent]
            if case["top"]:
                # of equal values the one with the lowest index: by rank, then by index
                rank = torch.unique(z, return_inverse=True)[1]
                order = rank * case["V"] + (case["V"] - 1 - torch.arange(case["V"], device=dev))
                ids = torch.topk(order, case["top"]).indices
                out += [ids, lp.gather(1, ids)]
            if kind == "score_grad":
                a = s["dlogprobs"][r:r + 512, None].double() * given[:, None]
                b = s["dentropy"][r:r + 512, None].double()
                hot = torch.zeros_like(z)
                hot[torch.arange(len(t), device=dev), t * given] = 1.0
                out.append(a * (hot - p) - b * (p * (lp + ent[:, None])).nan_to_num(0.0))
            outs.append(out)
        return tuple(torch.cat(o) for o in zip(*outs))
    g = torch.Generator(device=dev).manual_seed(seed)
    if kind == "linear4":
        w = (0.02 * torch.randn(case["N"], case["K"], generator=g, device=dev)).to(dt)
        x = torch.randn(case["M"], case["K"], generator=g, device=dev).to(dt).double()
        return x @ _decoded64(w, case["group"]).t()
    B, L, Hkv, D, S = (case[n] for n in ("B", "L", "Hkv", "D", "S"))
    k = _head_rows((B, Hkv, S, D), g, dev, dt)
    v = _head_rows((B, Hkv, S, D), g, dev, dt)
    if kind == "cache_write":
        kv = torch.randn(B, L, 2 * Hkv, D, generator=g, device=dev).to(dt)
        outs = []
        for old, new in ((k, kv[:, :, :Hkv]), (v, kv[:, :, Hkv:])):
            rows = torch.empty(B, Hkv, L, D, dtype=torch.float64, device=dev)
            for b, (start, count) in enumerate(zip(_starts(case), _counts(case))):
                rows[b] = old[b, :, start:start + L].double()
                rows[b, :, :count] = new[b, :count].transpose(0, 1).double()
                rows[b] = _decoded64(rows[b], CACHE_GROUP)
            outs.append(rows)
        return tuple(outs)
    q = (2 * torch.randn(B, L, case["Hq"], D, generator=g, device=dev)).to(dt).transpose(1, 2)
    return _attend64(case, dict(q=q), k, v)
