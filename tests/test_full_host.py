"""Attention over full-width pages and eviction without a GPU: the oracle against the definitions, the
host geometry, and every refusal of the entry points. No kernel is launched here."""

import ctypes
import math

import numpy as np
import pytest
import torch

from everserve_amd import kernels
from everserve_amd.state.evict import Evictor
from everserve_amd.state.full import FullCache, SharedPrefix
from oracle import full

FAKE = ctypes.c_void_p(1 << 20)  # never dereferenced: each call stops at its checks


@pytest.fixture(scope="module")
def lib():
    return kernels.open_library(kernels.library_path())


@pytest.fixture(scope="module")
def shim(lib):
    return kernels.Kernels(lib, kernels.library_path())


def message(lib, rc):
    assert rc == 1
    return lib.evs_last_error().decode()


# ---------------------------------------------------------------- the oracle
def test_a_prefix_and_own_tokens_are_one_context():
    g = np.random.default_rng(1)
    view = g.standard_normal((9, 4, 2, 2, 8))
    q = g.standard_normal((3, 4, 8))
    # two sequences behind 8 tokens, with pages of their own; and the same as whole contexts
    split = full.attend(q, view, np.array([[2], [3]]), [3, 2], [0, 1, 3], 0.4,
                        (np.array([[0, 1]]), [8], [0, 2]))
    whole = full.attend(q, view, np.array([[0, 1, 2], [0, 1, 3]]), [11, 10], [0, 1, 3], 0.4)
    assert np.allclose(split["out"], whole["out"]) and np.allclose(split["lse"], whole["lse"])
    # against the softmax written out for one row
    k, v = view[[0, 1, 2]].reshape(12, 2, 2, 8)[:11, 1].transpose(1, 0, 2)
    s = np.exp(0.4 * k @ q[0, 2])
    assert np.allclose(whole["out"][0, 2], s @ v / s.sum())


def test_weights_of_a_step_are_one_of_each_row_and_new_tokens_start_afresh():
    g = np.random.default_rng(2)
    view = g.standard_normal((9, 4, 2, 2, 8))
    q = g.standard_normal((4, 6, 8))
    mass = g.random((9, 2, 4))
    old = mass.copy()
    r = full.attend(q, view, np.array([[2], [3]]), [3, 2], [0, 2, 4], 0.4,
                    (np.array([[0, 1]]), [7], [0, 2]), mass)
    assert math.isclose(r["gave"].sum(), 4 * 6) and not r["gave"][1, :, 3].any()
    fresh = [(2, 1), (2, 2), (3, 0), (3, 1)]
    for p, o in fresh:
        assert np.array_equal(mass[p, :, o], r["gave"][p, :, o])
        old[p, :, o] = 0
    assert np.allclose(mass, old + r["gave"])


def test_the_choice_keeps_the_newest_and_the_heaviest():
    mass = np.array([[5.0, 1, 3, 3], [3, 0, 9, 2]])
    tables = [0, 1]
    assert full.choose(mass, tables, 8, 8, 2, 2) == list(range(8))
    assert full.choose(mass, tables, 8, 4, 1, 2) == [0, 2, 6, 7]
    assert full.choose(mass, tables, 8, 4, 0, 2) == [0, 2, 3, 6]  # of equal ones the first
    assert full.choose(mass, tables, 8, 3, 3, 2) == [5, 6, 7]
    assert full.choose(mass, [0, 5], 8, 5, 1, 2) == [0, 1, 2, 3, 7]  # a page that is none: last
    mass[0, 1], mass[1, 1], mass[0, 0] = math.nan, -0.0, 0.0
    assert full.choose(mass, tables, 8, 2, 0, 2) == [1, 6]
    mass[:] = 0
    mass[0, 2] = -0.0
    assert full.choose(mass, tables, 8, 3, 0, 2) == [0, 1, 2]


# ---------------------------------------------------------------- geometry
@pytest.mark.parametrize("layout,shape", [("kv_first", (2, 7, 16, 3, 80)),
                                          ("blocks_first", (7, 2, 16, 3, 80)),
                                          ("combined", (7, 3, 16, 160))])
def test_a_cache_knows_its_geometry(layout, shape):
    c = FullCache(torch.zeros(shape, dtype=torch.bfloat16))
    assert (c.layout.value, c.num_blocks, c.block_size, c.num_heads, c.head_dim) == (
        layout, 7, 16, 3, 80)
    e = Evictor([c.tensor, c.tensor.clone()])
    assert (e.num_blocks, e.block_size, e.num_heads, e.head_dim) == (7, 16, 3, 80)
    two = (2,) + shape[1:] if layout != "kv_first" else (2, 2) + shape[2:]
    named = FullCache(torch.zeros(two, dtype=torch.float16), layout)
    assert (named.layout.value, named.num_blocks) == (layout, 2)


def test_tensors_that_are_no_cache_are_refused():
    good = torch.zeros(7, 2, 16, 3, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="bf16 or f16"):
        FullCache(good.float())
    with pytest.raises(ValueError, match="kv_first"):
        FullCache(good, "kv_first")
    with pytest.raises(ValueError, match="combined"):
        FullCache(good, "combined")
    with pytest.raises(ValueError, match="layout"):
        FullCache(good[0, 0])
    for d in (8, 60, 264):
        with pytest.raises(ValueError, match="head size"):
            FullCache(torch.zeros(7, 2, 16, 3, d, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="16 bytes"):
        FullCache(torch.zeros(7, 2, 16, 3, 68, dtype=torch.bfloat16)[..., :64])
    with pytest.raises(ValueError, match="16 bytes"):
        FullCache(torch.zeros(good.numel() + 8, dtype=torch.bfloat16)[4:-4].view(good.shape))
    with pytest.raises(ValueError, match="16 bytes"):
        FullCache(torch.zeros(7, 2, 16, 3, 128, dtype=torch.bfloat16)[..., ::2])
    with pytest.raises(ValueError, match="contiguous"):
        Evictor([torch.zeros(7, 2, 16, 3, 128, dtype=torch.bfloat16)[..., ::2]])


# ---------------------------------------------------------------- the entry points' refusals
def strides(*s):
    return (ctypes.c_int64 * 5)(*s)


GOOD = strides(16 * 2 * 64, 2 * 64, 64, 9 * 16 * 2 * 64, 1)


def test_the_attention_call_refuses_what_it_cannot_do(lib):
    def attend(type_=0, out=FAKE, tokens=3, q_heads=4, heads=2, d=64, st=GOOD, starts=None, seqs=3,
               max_q=1, scale=0.125, q=FAKE, lens=FAKE, tables=FAKE, width=5, work=None, size=0,
               max_len=0, cache=FAKE, blocks=9, bs=16, pt=FAKE, pw=4, pl=FAKE, gs=FAKE, groups=1,
               max_prefix=0, qs=(256, 64), mass=None):
        return lib.evs_attend(q, (ctypes.c_int64 * 2)(*qs), type_, out, None, tokens, q_heads,
                              cache, blocks, bs, heads, d, st, tables, 5, width, lens, starts, seqs,
                              max_q, max_len, pt, 4, pw, pl, gs, groups, max_prefix, mass, scale,
                              work, size, None)

    assert "bf16 or f16" in message(lib, attend(type_=2))
    for d in (0, 8, 60, 264, -64):
        assert "head size" in message(lib, attend(d=d))
    for bad in (dict(blocks=-1), dict(bs=0), dict(heads=0), dict(blocks=1 << 31),
                dict(bs=1 << 31), dict(heads=1 << 16)):
        assert "bad cache" in message(lib, attend(**bad))
    for bad in (dict(width=-1), dict(pw=-1), dict(width=1 << 31)):
        assert "table width" in message(lib, attend(**bad))
    for bad in (dict(q_heads=5), dict(q_heads=0), dict(seqs=-1), dict(tokens=-1), dict(max_q=-1),
                dict(max_len=-1), dict(max_prefix=-1), dict(groups=-1), dict(tokens=1 << 31),
                dict(tokens=1 << 30)):
        assert "bad count" in message(lib, attend(**bad))
    for scale in (0.0, -1.0, math.inf, math.nan, 3e38):
        assert "scale" in message(lib, attend(scale=scale))
    assert "five strides" in message(lib, attend(st=None))
    assert "contiguous" in message(lib, attend(st=strides(2048, 128, 64, 18432, 2)))
    for at in range(4):
        s = list(GOOD)
        s[at] += 4
        assert "rows must start on 16" in message(lib, attend(st=strides(*s)))
    assert "rows must start on 16" in message(lib, attend(cache=ctypes.c_void_p((1 << 20) + 8)))
    assert "one query a sequence" in message(lib, attend(tokens=4))
    assert "one query a sequence" in message(lib, attend(max_q=2))
    for name in ("q", "lens", "tables", "cache", "out", "pt", "pl", "gs"):
        assert "null" in message(lib, attend(**{name: None})), name
    assert "out must" in message(lib, attend(out=ctypes.c_void_p((1 << 20) + 8)))
    assert "queries must" in message(lib, attend(q=ctypes.c_void_p((1 << 20) + 8)))
    assert "queries must" in message(lib, attend(qs=(260, 64)))
    assert "queries must" in message(lib, attend(qs=(256, 68)))
    assert "too many" in message(lib, attend(tokens=1 << 23, seqs=1 << 23, groups=0))
    assert "to weigh" in message(lib, attend(tokens=1 << 19, seqs=1 << 19, q_heads=8, heads=8,
                                             groups=0, mass=FAKE))
    assert "workspace" in message(lib, attend())  # a prefix's parts are joined
    assert "workspace" in message(lib, attend(size=1 << 30))
    assert "workspace" in message(lib, attend(size=1 << 30, work=ctypes.c_void_p((1 << 20) + 8)))
    assert attend(tokens=0, q=None) == 0 and attend(seqs=0) == 0 and attend(max_q=0) == 0


def test_the_workspace_is_what_its_counts_need(lib):
    def need(seqs=4, tokens=4, q_heads=8, heads=2, d=64, max_q=1, max_len=1000, groups=0,
             max_prefix=0, mass=0):
        got = ctypes.c_int64(-1)
        rc = lib.evs_attend_workspace(seqs, tokens, q_heads, heads, d, max_q, max_len, groups,
                                      max_prefix, mass, ctypes.byref(got))
        return got.value if rc == 0 else message(lib, rc)

    assert need(max_len=16) == 0  # one part a row: it is written where it goes
    # a reference, the running maximum and sum, and 16 scores for each of 4 x 8 rows
    assert need(max_len=16, mass=1) == 4 * 8 * (4 + 8 + 16 * 4)
    assert need(max_len=16, groups=1, max_prefix=16) == 2 * 4 * 8 * (64 + 2) * 4
    assert need(max_len=100000) > 0
    assert need(seqs=0, tokens=0) == 0 and need(max_q=0) == 0
    assert "bad count" in need(q_heads=7)
    assert "bad count" in need(d=60)
    assert lib.evs_attend_workspace(1, 1, 1, 1, 64, 1, 1, 0, 0, 0, None) == 1
    # longer contexts never need parts without end: 1,024 of a context, 4,096 workgroups of a kind
    assert need(max_len=(1 << 31) - 1, groups=1, max_prefix=(1 << 31) - 1) <= (
        (1024 + 4096 // 8) * 4 * 8 * (64 + 2) * 4)


def test_the_eviction_call_refuses_what_it_cannot_do(lib):
    def evict(layers=2, blocks=9, heads=2, d=64, bs=16, st=strides(2048, 128, 64, 18432, 1), elem=2,
              tables=FAKE, width=5, lens=FAKE, seqs=3, new=FAKE, new_width=3, budget=40, recent=4,
              mass=FAKE, out=FAKE, kept=FAKE, ptrs=FAKE):
        return lib.evs_evict(ptrs, layers, blocks, heads, d, bs, st, elem, tables, 5, width, lens,
                             seqs, new, 3, new_width, budget, recent, mass, out, kept, None)

    assert "five strides" in message(lib, evict(st=None))
    assert "element size" in message(lib, evict(elem=8))
    for bad in (dict(layers=0), dict(layers=70000), dict(blocks=-1), dict(heads=0), dict(d=0),
                dict(d=1 << 16), dict(bs=0), dict(heads=1 << 16)):
        assert "bad caches" in message(lib, evict(**bad))
    for bad in (dict(width=-1), dict(seqs=-1), dict(width=1 << 28), dict(new_width=-1)):
        assert "bad tables" in message(lib, evict(**bad))
    for bad in (dict(budget=-1, recent=0), dict(budget=(1 << 31) - 1024), dict(recent=41), dict(recent=-1)):
        assert "newest" in message(lib, evict(**bad))
    assert "hold no" in message(lib, evict(budget=49))
    assert "contiguous" in message(lib, evict(st=strides(2048, 128, 64, 18432, 2)))
    assert "stride" in message(lib, evict(st=strides(2048, 0, 64, 18432, 1)))
    for name in ("tables", "lens", "new", "mass", "out", "kept", "ptrs"):
        assert "null" in message(lib, evict(**{name: None})), name
    assert "layers, sequences" in message(lib, evict(layers=65535, seqs=65535))
    assert "tiles of rows" in message(lib, evict(layers=1, heads=1, seqs=1 << 20, new_width=1 << 16,
                                                 budget=1 << 20, bs=16))
    assert evict(seqs=0, lens=None) == 0


def test_the_shim_refuses_host_tensors_and_wrong_shapes(shim):
    t = torch.zeros(4, 2, 16, 2, 64, dtype=torch.bfloat16)
    c = FullCache(t)
    q, tables, lens = torch.zeros(1, 4, 64).bfloat16(), torch.zeros(1, 2).int(), torch.ones(1).int()
    with pytest.raises(RuntimeError, match="on the device"):
        shim.attend(q, t, 4, 16, 2, c.strides, tables, lens)
    with pytest.raises(RuntimeError, match="bf16 or f16|bf16 "):
        shim.attend(q.float(), t, 4, 16, 2, c.strides, tables, lens)
    with pytest.raises(ValueError, match="expected"):
        c.attend(q[..., :32], tables, lens)
    with pytest.raises(RuntimeError, match="on the\\s+device"):
        shim.evict(torch.zeros(1).long(), 4, 2, 64, 16, c.strides, 2, tables, lens, tables, 16,
                   torch.zeros(1, 4, 2, 16))
    p = SharedPrefix(tables, lens, torch.zeros(2).int())
    assert p.max_len == 0
