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


# where a wave's lanes write what its other lanes read
EXCHANGES = [("full_rows.hpp", "lds.at[wave]"), ("full_weigh.hip", "s_query[wave]"),
             ("full_weigh.hip", "s_sum[wave]")]
SYNC = re.compile(r"\b(wave_sync|__syncthreads)\(\);")


@pytest.mark.parametrize("name,array", EXCHANGES, ids=lambda x: x.split("[")[0])
def test_a_waves_writes_stand_between_waits_of_it(name, array):
    """Those ahead for the reads of what was there before, those behind for the reads of them."""
    text = code_of(next(p for p in SOURCES if p.name == name).read_text())
    stores = [m.start() for m in re.finditer(re.escape(array) + r"[^;{}]*\]\s*=[^=]", text)]
    assert len(stores) == 1
    before = [m.end() for m in SYNC.finditer(text, 0, stores[0])]
    behind = SYNC.search(text, stores[0])
    assert before and behind
    between = text[before[-1]:behind.start()]
    assert between.count(array) == 1, between  # the store alone


def test_a_barrier_without_one_is_found():
    bare = "s[lane] = x;\n  __builtin_amdgcn_wave_barrier();  // read by others\n  y = s[0];"
    assert unfenced(bare) == ["s[lane] = x"]
    fenced = bare.replace("  __b", '  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");\n  __b')
    assert unfenced(fenced) == []
