"""CPU: calls of the serving side at their limits, through the C ABI with addresses
that are never read or with the GPU's part replaced, and what its kernels' sources
have to keep to."""
import ctypes
import os
import re

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "elastic-sparse-attention_b200", "csrc")


# ---------------------------------------------------------------------------
# A kernel that may start while the kernel before it still writes reads what that one
# wrote with ordinary loads: those of the read-only path want memory that does not
# change while the kernel runs.
# ---------------------------------------------------------------------------
READ_ONLY = re.compile(r"__ldg\b|\bldg16\b|\bldg16_stream\b|\.nc\b")


def functions(source):
    """{name: text} of the functions of a source file; a function's text begins at its
    name (its declaration's templates and qualifiers are not looked at)."""
    source = re.sub(r"//[^\n]*", "", source)
    found = {}
    for m in re.finditer(r"\b(\w+)\s*\((?:[^()]|\([^()]*\))*\)\s*(?:const\s*)?\{", source):
        if m[1] in ("if", "for", "while", "switch", "constexpr"):
            continue
        depth, i = 0, m.end() - 1
        while True:
            depth += {"{": 1, "}": -1}.get(source[i], 0)
            i += 1
            if depth == 0:
                break
        found.setdefault(m[1], "")
        found[m[1]] += source[m.start():i]
    return found


def early_read_only_loads(source):
    """(kernel, function) of read-only loads in the kernels that wait for the one before
    them, and in the functions of the file that they call."""
    all_ = functions(source)
    bad = []
    for name, text in all_.items():
        if "cudaGridDependencySynchronize" not in text:
            continue
        todo, seen = [name], set()
        while todo:
            f = todo.pop()
            if f in seen:
                continue
            seen.add(f)
            if READ_ONLY.search(all_[f]):
                bad.append((name, f))
            todo += [w for w in set(re.findall(r"\b(\w+)\s*(?:<[\w, ]*>)?\(", all_[f])) if w in all_]
    return bad


def test_the_check_sees_read_only_loads():
    text = ("int help(const int* p) {{ return {}(p); }}\n"
            "__global__ void k(const int* p) {{\n  cudaGridDependencySynchronize();\n  help(p);\n}}\n"
            "__global__ void other(const int* p) {{ __ldg(p); }}\n")
    assert early_read_only_loads(text.format("__ldg")) == [("k", "help")]
    assert early_read_only_loads(text.format("load")) == []


@pytest.mark.parametrize("name", ["esa_score.cuh", "esa_weight4.cuh"])
def test_kernels_that_start_early_read_with_ordinary_loads(name):
    with open(os.path.join(CSRC, name)) as f:
        source = f.read()
    waiting = [k for k, t in functions(source).items() if "cudaGridDependencySynchronize" in t]
    assert waiting
    assert early_read_only_loads(source) == []


def session_without_a_gpu(esa, batch, vocab=50):
    s = object.__new__(esa.PackedDecoder)
    s.lengths = torch.zeros(batch, dtype=torch.int64)
    s.lm_head = esa.layer_ops.PackedWeight4(None, None, (vocab, 64), 32, torch.bfloat16)
    return s


@pytest.mark.parametrize("pad", [-1, -100, 50, 1 << 40])
def test_ids_of_padding_are_not_looked_up(esa, pad):
    """Whatever a padded place holds, the embedding sees an id of the vocabulary there
    (its lookup on the GPU does not survive another one)."""
    class Seen(Exception):
        pass

    class Stack:
        Hq, Hkv, D, hidden, eps = 1, 1, 64, 64, 1e-6

        def _embed(self, ids):
            raise Seen(ids)

    s = session_without_a_gpu(esa, 3)
    s.stack = Stack()
    ids = torch.tensor([[1, 2, 3], [4, pad, pad], [pad, pad, pad]])
    given = ids.clone()
    for call in (s.step, s.score):
        with pytest.raises(Seen) as e:
            call(ids, torch.tensor([3, 1, 0]))
        assert e.value.args[0].tolist() == [[1, 2, 3], [4, 0, 0], [0, 0, 0]]
        assert torch.equal(ids, given)
        with pytest.raises(Seen) as e:
            call(ids, None)
        assert torch.equal(e.value.args[0], ids)                  # without counts all are tokens


@pytest.mark.parametrize("top_k,vocab", [(33, 50), (-1, 50), (8, 7)])
def test_scores_refuse_top_k_before_the_tokens_are_fed(esa, monkeypatch, top_k, vocab):
    """A refused call leaves the sequences as they were."""
    s = session_without_a_gpu(esa, 2, vocab)
    fed = []
    monkeypatch.setattr(esa.PackedDecoder, "step", lambda *a: fed.append(a))
    with pytest.raises(ValueError, match="top_k"):
        s.score(torch.zeros(2, 3, dtype=torch.int64), top_k=top_k)
    assert not fed and not s.lengths.any()


# ---------------------------------------------------------------------------
# empty and refused calls
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("name", ["write", "read", "forward"])
def test_a_cache_of_no_sequences(esa, name):
    """Its tensors have no memory; there is nothing to do."""
    lib = esa._lib.load()
    none = esa._lib.EsaTensor(None, 0, 64, 64)
    c = esa._lib.EsaCache4(None, None, 0, 2, 64, 0, 100)
    c = ctypes.byref(c)
    if name == "write":
        rc = lib.esa_cache4_write(1, c, 4, none, none, None, 0, None, None)
    elif name == "read":
        rc = lib.esa_cache4_read(1, c, 4, none, none, None, 0, None)
    else:
        rc = lib.esa_cache4_forward(1, c, 4, 4, 16, 1, 4, 0, 0, 0.1, none, None, 0, None, none, None,
                                    None)
    assert rc == 0, lib.esa_last_error()


@pytest.mark.parametrize("shape", [(1, 12), (3, 4), (12,), (2, 7)])
def test_scores_refuse_labels_of_another_shape(esa, shape):
    """As many labels in another shape would be paired with other rows."""
    stack = object.__new__(esa.ElasticDecoderStack)
    with pytest.raises(ValueError, match="labels"):
        esa.ElasticDecoderStack.token_logprobs(stack, torch.zeros(2, 6, dtype=torch.int64),
                                               torch.zeros(shape, dtype=torch.int64))
