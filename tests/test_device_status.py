"""The words that a kernel may leave in the device status: one value per condition, kept as they are (joined by OR, 0x..09 and 0x..0A read as 0x..0B)."""
import pathlib
import re

CSRC = pathlib.Path(__file__).resolve().parents[1] / "webgpu_b200" / "csrc"
SOURCES = {f.name: f.read_text() for f in sorted(CSRC.glob("*.cu")) + sorted(CSRC.glob("*.cuh"))}


def test_one_value_per_condition():
    words = re.findall(r"constexpr uint32_t (STATUS_\w+) = (0x[0-9A-Fa-f]+)u;", SOURCES["common.cuh"])
    assert len(words) >= 10 and len({int(v, 16) for _, v in words}) == len(words)
    for name, text in SOURCES.items():                         # and none defined elsewhere
        code = re.sub(r"//.*", "", text)
        assert name == "common.cuh" or not re.search(r"0x7C05[0-9A-Fa-f]{4}", code), name


def test_words_are_not_joined():
    for name, text in SOURCES.items():
        assert not re.search(r"atomic\w+\((?:\w+(?:\.|->))?status\b", text.replace("atomicCAS(status, 0u, code)", "")), name
