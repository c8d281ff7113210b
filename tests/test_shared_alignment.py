"""Static shared arrays that kernels read or write 16 bytes at a time say that they start on 16 bytes (from the sources, host
only): without it the compiler may put them anywhere their elements' type allows."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "from_scratch_inference_engine_b200" / "csrc"
FILES = sorted(p for p in CSRC.iterdir() if p.suffix in (".cu", ".cuh"))
DECLARED = re.compile(r"^[ \t]*(?:static )?__shared__\s+(alignas\(\d+\)\s+|__align__\(\d+\)\s+)?([A-Za-z_][\w:]*(?:<[^;=]*?>)?)\s+([^;(]+);", re.M)
WIDE_TYPES = ("float4", "uint4", "int4", "double2", "ulonglong2", "longlong2")
WIDE = r"(?:reinterpret_cast<\s*(?:const\s+)?(?:%s)\s*\*>\(\s*|(?:load|store)_cols\(\s*)&?\(?%%s\b" % "|".join(WIDE_TYPES)


def kernels(text):
    """The text cut where a kernel or function begins: a name means an array of the same piece."""
    cuts = [m.start() for m in re.finditer(r"^(?:template|__global__|__device__|static|inline)\b", text, re.M)] + [len(text)]
    return [text[a:b] for a, b in zip([0] + cuts, cuts)]


def unaligned(text):
    found = []
    for piece in kernels(text):
        for aligned, kind, names in DECLARED.findall(piece):
            if aligned or kind in WIDE_TYPES:
                continue
            for name in re.findall(r"([A-Za-z_]\w*)\s*(?=\[)", re.sub(r"\[[^\]]*\]", "[]", names)):
                if re.search(WIDE % re.escape(name), piece):
                    found.append(name)
    return found


def test_the_search_finds_what_it_looks_for():
    """Planted in a text, not in a kernel."""
    plain = "__global__ void k() {\n    __shared__ float a[2][8], b[4];\n    x = *reinterpret_cast<const float4*>(&%s[0][0]);\n}\n"
    assert unaligned(plain % "a") == ["a"] and unaligned(plain % "b") == ["b"] and unaligned(plain % "c") == []
    assert unaligned((plain % "a").replace("float a", "__align__(16) float a")) == []
    assert unaligned("__global__ void k() {\n    __shared__ float s[4];\n    store_cols(&s[0], v);\n}\n") == ["s"]


@pytest.mark.parametrize("path", FILES, ids=lambda p: p.name)
def test_wide_accesses_are_to_aligned_arrays(path):
    assert unaligned(path.read_text()) == []
