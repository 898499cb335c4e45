"""A static shared array that a kernel also accesses through a wider type must
be declared with that type's alignment: nothing else places it on such a border."""
import glob
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
WIDTH = {"uint2": 8, "uint4": 16, "float2": 8, "float4": 16, "uint32_t": 4, "int": 4, "float": 4,
         "uint64_t": 8}
BASE = {"uint8_t": 1, "uint16_t": 2, "uint32_t": 4, "int": 4, "float": 4, "float4": 16,
        "uint4": 16, "uint64_t": 8}


def misaligned(source):
    """(array, declared alignment, access width) of each wider access."""
    bad = []
    declared = re.compile(r"__shared__\s+(?:__align__\((\d+)\)\s+)?(\w+)\s+(\w+)\[")
    for m in declared.finditer(source):
        align, type_, name = int(m[1] or 0) or BASE[m[2]], m[2], m[3]
        end = source.find("\n}\n", m.end())          # of the function it is declared in
        body = source[m.end():end if end >= 0 else len(source)]
        for cast in re.finditer(r"reinterpret_cast<(?:const )?(\w+)\s*\*>\(\s*&?" + name + r"\b", body):
            if WIDTH[cast[1]] > align:
                bad.append((name, align, WIDTH[cast[1]]))
    return bad


def test_the_check_sees_a_narrow_declaration():
    text = "__global__ void k() {{\n  __shared__ {}uint16_t cnt[4][8];\n  reinterpret_cast<uint32_t*>(&cnt[0][0])[1] = 0;\n}}\n"
    assert misaligned(text.format("")) == [("cnt", 2, 4)]
    assert misaligned(text.format("__align__(4) ")) == []


def test_shared_arrays_are_aligned_for_their_accesses():
    files = sorted(glob.glob(os.path.join(ROOT, "elastic-sparse-attention_b200", "csrc", "*.cu*")))
    assert files
    bad = {}
    for f in files:
        with open(f) as fh:
            text = re.sub(r"extern __shared__[^;]*;", "", fh.read())
        if found := misaligned(text):
            bad[os.path.basename(f)] = found
    assert not bad, bad
