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
    # an array that a vector is copied through: *reinterpret_cast<vector*>(name) with the name of a local array
    arrays = re.findall(r"^\s*((?:alignas\(\d+\) )?)(?:T|float|double|uint32_t) (\w+)\[[^;]*;", text, re.M)
    vectors = set(re.findall(r"reinterpret_cast<(?:const )?(?:u?int[24]|float[24]|W|typename Bits<[^;]*>::type)\s*\*>\((\w+)\)", text))
    for align, name in arrays:
        if name in vectors:
            assert align == "alignas(16) ", (file.name, name)


@pytest.mark.parametrize("file", FILES, ids=lambda f: f.name)
def test_dynamic_shared_memory_is_aligned(file):
    for align, kind, name in re.findall(r"extern __shared__ ((?:__align__\(\d+\) )?)([\w ]+?) (\w+)\[\];", file.read_text()):
        if kind == "uint32_t":                                 # plain words (the lengths of a plan)
            continue
        if f"(smem_u32({name}) & 1023u)" in file.read_text():  # moved up to a boundary by hand
            continue
        assert align, (file.name, name)
