"""What lanes of a wave pass to each other through LDS, in the sources: a wave's barrier orders no
memory by itself, so each stands behind a fence of the wavefront."""

import re
from pathlib import Path

import pytest

import everserve_amd

SOURCES = sorted(p for p in (Path(everserve_amd.__file__).parent / "csrc").iterdir()
                 if p.suffix in (".hip", ".hpp"))


def code_of(text: str) -> str:
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", text, flags=re.S)


def unfenced(text: str) -> list:
    """The statements ahead of the wave barriers that are no fence of theirs."""
    parts = code_of(text).split("__builtin_amdgcn_wave_barrier()")
    before = [p.rstrip().rstrip(";").rstrip() for p in parts[:-1]]
    fence = re.compile(
        r'__builtin_amdgcn_fence\(__ATOMIC_(RELEASE|ACQ_REL|SEQ_CST), "wavefront"\)$')
    return [b.splitlines()[-1].strip() for b in before if not fence.search(b)]


@pytest.mark.parametrize("path", SOURCES, ids=lambda p: p.name)
def test_a_waves_barrier_stands_behind_a_fence(path):
    assert unfenced(path.read_text()) == []


def test_a_barrier_without_one_is_found():
    bare = "s[lane] = x;\n  __builtin_amdgcn_wave_barrier();  // read by others\n  y = s[0];"
    assert unfenced(bare) == ["s[lane] = x"]
    fenced = bare.replace("  __b", '  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");\n  __b')
    assert unfenced(fenced) == []
