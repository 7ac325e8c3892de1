"""Places that the kernels of a paged KV cache reach by whole vectors, cp.async or bulk copies are declared with the alignment these need: an access
of 16 bytes at an address that only happens to be aligned is a misaligned one as soon as the compiler lays things out otherwise."""
import pathlib
import re

import pytest

CSRC = pathlib.Path(__file__).resolve().parents[1] / "webgpu_b200" / "csrc"
FILES = sorted(CSRC.glob("paged_*.cu")) + sorted(CSRC.glob("paged*.cuh")) + [CSRC / "verify_drafts.cu"]


@pytest.mark.parametrize("file", FILES, ids=lambda f: f.name)
def test_arrays_that_vectors_go_through_are_aligned(file):
    text = file.read_text()
    # an array that a vector is copied through, *reinterpret_cast<vector*>(its name), within the lines behind its declaration
    for found in re.finditer(r"^\s*((?:alignas\(\d+\) )?)T (\w+)\[[^;]*;", text, re.M):
        vector = r"reinterpret_cast<(?:const )?(?:u?int[24]|float[24]|uint32_t|W|typename Bits<[^;]*>::type)\s*\*>\(%s\)" % found[2]
        if re.search(vector, text[found.end():found.end() + 600]):
            assert found[1] == "alignas(16) ", (file.name, found[2])


@pytest.mark.parametrize("file", FILES, ids=lambda f: f.name)
def test_dynamic_shared_memory_is_aligned(file):
    for align, kind, name in re.findall(r"extern __shared__ ((?:__align__\(\d+\) )?)([\w ]+?) (\w+)\[\];", file.read_text()):
        if kind == "uint32_t":                                 # plain words (the lengths of a plan)
            continue
        if f"(smem_u32({name}) & 1023u)" in file.read_text():  # moved up to a boundary by hand
            continue
        assert align, (file.name, name)
