"""The 4-bit cache and the page moves without a GPU: the oracle against the definitions, the host
geometry, and every refusal of the entry points. No kernel is launched here."""

import ctypes
import math

import numpy as np
import pytest
import torch

from everserve_amd import kernels
from everserve_amd.state.fp4 import Fp4Cache, cache_shape, row_bytes
from everserve_amd.state.pages import PageMover
from everserve_amd.state.paged import PagedKV
from oracle import fp4

FAKE = ctypes.c_void_p(1 << 20)  # never dereferenced: each call stops at its checks


@pytest.fixture(scope="module")
def lib():
    return kernels.open_library(kernels.library_path())


@pytest.fixture(scope="module")
def shim(lib):
    return kernels.Kernels(lib, kernels.library_path())


# ---------------------------------------------------------------- the oracle
def test_every_code_survives_a_round_trip():
    for e in (-126, -20, 0, 3, 125):
        x = np.concatenate((fp4.GRID, -fp4.GRID, fp4.GRID, -fp4.GRID)) * 2.0 ** e
        byte, codes = fp4.encode_group(x)
        assert byte == e + 127
        half = fp4.encode(x)
        assert np.array_equal(fp4.decode(half, 32), x)
        assert np.array_equal(np.signbit(fp4.decode(half, 32)), np.signbit(x))


def test_codes_are_the_nearest_and_ties_go_to_the_even_code():
    x = np.zeros(32)
    x[0] = 6
    edges = {0.25: 0, 0.75: 1, 1.25: 1, 1.75: 2, 2.5: 2, 3.5: 4, 5: 4}
    for i, v in enumerate(edges):
        x[1 + i] = v
        x[10 + i] = np.nextafter(v, 9)
        x[20 + i] = np.nextafter(v, 0)
    got = fp4.decode(fp4.encode(x), 32)
    for i, (v, want) in enumerate(edges.items()):
        assert got[1 + i] == want
        assert got[10 + i] > v > got[20 + i]


def test_the_scale_is_the_least_that_brings_the_largest_to_seven():
    for most, e in ((7.0, 0), (np.nextafter(7.0, 8), 1), (3.5, -1), (3.6, 0), (0.0, -126),
                    (2.0 ** -140, -126), (3.38e38, 125)):
        x = np.zeros(8)
        x[3] = -most
        assert fp4.encode_group(x)[0] == e + 127, most
    for bad in (math.inf, -math.inf, math.nan):
        x = np.ones(40)
        x[35] = bad
        half = fp4.encode(x)
        got = fp4.decode(half, 40)
        assert np.all(got[:32] == 1) and np.all(np.isnan(got[32:]))


def test_the_error_of_a_held_row_is_half_a_step():
    rng = np.random.default_rng(5)
    x = rng.standard_normal((50, 128)) * np.exp2(rng.integers(-10, 10, (50, 1)))
    got = fp4.decode(fp4.encode(x), 128)
    most = np.abs(x.reshape(50, 4, 32)).max(-1).repeat(32, -1).reshape(50, 128)
    # the widest step is 2 scales, and a scale is at most 2/7 of the group's largest magnitude
    assert np.all(np.abs(got - x) <= 2 / 7 * most)


def test_a_plan_moves_each_page_past_the_front_into_one_hole():
    rng = np.random.default_rng(6)
    for _ in range(50):
        blocks = int(rng.integers(1, 60))
        tables = rng.integers(-2, blocks + 2, (5, 7))
        counts = rng.integers(-1, 8, 5)
        new, moves, used = fp4.plan_compaction(tables, counts, blocks)
        src, dst = {a for a, _ in moves}, {b for _, b in moves}
        assert not src & dst and len(src) == len(dst) == len(moves) <= blocks // 2
        named = {p for row, n in zip(new, counts) for p in row[:max(0, n)] if 0 <= p < blocks}
        assert named == set(range(used))


# ---------------------------------------------------------------- geometry
@pytest.mark.parametrize("d", range(16, 257, 8))
def test_a_half_rows_bytes_are_the_librarys(lib, d):
    got = ctypes.c_int64()
    assert lib.evs_fp4_row_bytes(d, ctypes.byref(got)) == 0
    assert got.value == row_bytes(d) == fp4.row_bytes(d) and got.value % 4 == 0


@pytest.mark.parametrize("d", [0, 8, 12, 100, 264, -16])
def test_other_head_sizes_are_refused(lib, d):
    with pytest.raises(ValueError, match="head size"):
        row_bytes(d)
    assert lib.evs_fp4_row_bytes(d, ctypes.byref(ctypes.c_int64())) == 1
    assert b"head size" in lib.evs_last_error()


@pytest.mark.parametrize("layout", ["kv_first", "blocks_first", "combined"])
def test_a_cache_knows_its_geometry_and_is_a_cache_of_bytes_to_the_rest(layout):
    c = Fp4Cache.empty(7, 16, 3, 80, layout, device="cpu")
    assert (c.num_blocks, c.block_size, c.num_heads, c.head_dim) == (7, 16, 3, 80)
    p = PagedKV.of(c.tensor)
    assert (p.layout.value, p.num_blocks, p.block_size, p.num_heads, p.head_dim) == (
        layout, 7, 16, 3, row_bytes(80))
    assert p.layout_strides(c.tensor) == c.strides
    two = Fp4Cache.empty(2, 16, 3, 80, layout, device="cpu")  # fits two layouts: the name decides
    assert (two.layout.value, two.num_blocks) == (layout, 2)
    mover = PageMover([c.tensor, c.tensor.clone()])
    assert (mover.num_blocks, mover.block_size, mover.num_heads) == (7, 16, 3)


def test_tensors_that_are_no_cache_are_refused():
    with pytest.raises(ValueError, match="uint8"):
        Fp4Cache(torch.zeros(cache_shape("combined", 3, 16, 2, 64)), 64)
    with pytest.raises(ValueError, match="shape"):
        Fp4Cache(torch.zeros(3, 2, 16, 2 * row_bytes(64), dtype=torch.uint8), 128)
    with pytest.raises(ValueError, match="shape"):
        Fp4Cache(torch.zeros(2, 3, 16, 2, 36, dtype=torch.uint8), 64, "combined")
    odd = torch.zeros(2, 3, 16, 2, 38, dtype=torch.uint8)[..., :36]  # rows off 4 bytes
    with pytest.raises(ValueError, match="4 bytes"):
        Fp4Cache(odd, 64)
    with pytest.raises(ValueError, match="no layers"):
        PageMover([])
    a = torch.zeros(4, 2, 16, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="one shape"):
        PageMover([a, a[:3]])
    with pytest.raises(ValueError, match="bytes"):
        PageMover([a.double()])
    with pytest.raises(ValueError, match="16-byte"):
        flat = torch.zeros(a.numel() + 8, dtype=torch.bfloat16)
        PageMover([flat[4:4 + a.numel()].view(a.shape)])
    with pytest.raises(ValueError, match="kv_first"):
        PageMover([a], "kv_first")


# ---------------------------------------------------------------- the entry points' refusals
def strides(*s):
    return (ctypes.c_int64 * 5)(*s)


GOOD = strides(16 * 2 * 2 * 36, 2 * 2 * 36, 2 * 36, 36, 1)


def message(lib, rc):
    assert rc == 1
    return lib.evs_last_error().decode()


def test_the_row_calls_refuse_what_they_cannot_address(lib):
    ins = (ctypes.c_int64 * 4)(128, 64, 128, 64)

    def write(key=FAKE, type_=0, n=4, cache=FAKE, blocks=9, bs=16, heads=2, d=64, st=GOOD,
              slots=FAKE):
        return lib.evs_fp4_write_rows(key, FAKE, ins, type_, slots, n, cache, blocks, bs, heads, d,
                                      st, None)

    def read(key=FAKE, n=4, type_=0, st=GOOD, d=64):
        return lib.evs_fp4_read_rows(FAKE, 9, 16, 2, d, st, FAKE, n, key, FAKE, type_, None)

    assert "element type" in message(lib, write(type_=3))
    assert "negative" in message(lib, write(n=-1))
    assert "head size" in message(lib, write(d=60))
    assert "five strides" in message(lib, write(st=None))
    assert "multiples of 4" in message(lib, write(st=strides(2306, 144, 72, 36, 1)))
    assert "multiples of 4" in message(lib, write(cache=ctypes.c_void_p((1 << 20) + 2)))
    assert "contiguous" in message(lib, write(st=strides(2304, 144, 72, 36, 2)))
    assert "bad cache" in message(lib, write(bs=0))
    assert "bad cache" in message(lib, write(heads=0))
    assert "bad cache" in message(lib, write(blocks=-1))
    assert "null" in message(lib, write(key=None))
    assert "null" in message(lib, write(slots=None))
    assert "null cache" in message(lib, write(cache=None))
    assert "off their element" in message(lib, write(key=ctypes.c_void_p((1 << 20) + 1)))
    assert write(n=0, key=None) == 0 and write(blocks=0, cache=None) == 0
    assert "16 bytes" in message(lib, read(key=ctypes.c_void_p((1 << 20) + 8)))
    assert "element type" in message(lib, read(type_=-1))
    assert "null" in message(lib, read(key=None))
    assert read(n=0, key=None) == 0


def test_the_attention_call_refuses_what_it_cannot_do(lib):
    qs = (ctypes.c_int64 * 2)(256, 64)

    def attend(type_=0, out=FAKE, tokens=3, q_heads=4, heads=2, d=64, st=GOOD, starts=None, seqs=3,
               max_q=1, scale=0.125, q=FAKE, lens=FAKE, tables=FAKE, width=5, work=None, size=0,
               max_len=0):
        return lib.evs_fp4_attend(q, qs, type_, out, None, tokens, q_heads, FAKE, 9, 16, heads, d,
                                  st, tables, 5, width, lens, starts, seqs, max_q, max_len, scale,
                                  work, size, None)

    assert "query type" in message(lib, attend(type_=2))
    assert "head size" in message(lib, attend(d=260))
    assert "query heads" in message(lib, attend(q_heads=5))
    assert "query heads" in message(lib, attend(q_heads=0))
    for scale in (0.0, -1.0, math.inf, math.nan):
        assert "scale" in message(lib, attend(scale=scale))
    assert "one query a sequence" in message(lib, attend(tokens=4))
    assert "one query a sequence" in message(lib, attend(max_q=2))
    assert "null" in message(lib, attend(q=None))
    assert "null" in message(lib, attend(lens=None))
    assert "null" in message(lib, attend(tables=None))
    assert "16 bytes" in message(lib, attend(out=ctypes.c_void_p((1 << 20) + 4)))
    assert "element size" in message(lib, attend(q=ctypes.c_void_p((1 << 20) + 1)))
    assert "bad count" in message(lib, attend(seqs=-1))
    assert "bad count" in message(lib, attend(width=-1))
    assert attend(tokens=0, q=None) == 0 and attend(seqs=0) == 0 and attend(max_q=0) == 0


def test_the_page_calls_refuse_what_they_cannot_do(lib):
    def copy(pairs=4, layers=2, blocks=9, heads=2, d=64, bs=16, st=strides(4096, 128, 64, 2048, 1),
             elem=2, src=FAKE, count=None):
        return lib.evs_copy_blocks(FAKE, layers, src, FAKE, pairs, count, blocks, heads, d, bs, st,
                                   elem, None)

    assert "element size" in message(lib, copy(elem=8))
    assert "five strides" in message(lib, copy(st=None))
    assert "negative" in message(lib, copy(pairs=-1))
    assert "layers" in message(lib, copy(layers=70000))
    assert "stride" in message(lib, copy(st=strides(4096, 128, -64, 2048, 1)))
    assert "null" in message(lib, copy(src=None))
    assert "words" in message(lib, copy(d=1 << 20, bs=1 << 20))
    assert "device count" in message(lib, copy(pairs=1 << 30, count=FAKE))
    for nothing in (dict(pairs=0), dict(layers=0), dict(blocks=0), dict(heads=0), dict(d=0),
                    dict(bs=0)):
        assert copy(src=None, **nothing) == 0

    def plan(rows=3, width=4, blocks=9, room=4, sizes=FAKE, work=FAKE, size=1 << 20, tables=FAKE):
        return lib.evs_plan_compaction(tables, rows, width, 4, None, blocks, FAKE, FAKE, FAKE,
                                       room, sizes, work, size, None)

    assert "room" in message(lib, plan(room=3))
    assert "workspace" in message(lib, plan(size=4))
    assert "workspace" in message(lib, plan(work=None))
    assert "workspace" in message(lib, plan(work=ctypes.c_void_p((1 << 20) + 2)))
    assert "null" in message(lib, plan(sizes=None))
    assert "null" in message(lib, plan(tables=None))
    assert "rows" in message(lib, plan(rows=-1))
    assert "pages" in message(lib, plan(blocks=-1))


def test_the_shim_refuses_host_tensors_and_wrong_shapes(shim):
    c = Fp4Cache.empty(4, 16, 2, 64, device="cpu")
    geo = (c.num_blocks, c.block_size)
    rows = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    slots = torch.arange(3)
    with pytest.raises(RuntimeError, match="on the device"):
        shim.fp4_write_rows(rows, rows, slots, c.tensor, *geo, c.strides)
    with pytest.raises(RuntimeError, match="shape"):
        shim.fp4_write_rows(rows, rows[:2], slots, c.tensor, *geo, c.strides)
    with pytest.raises(RuntimeError, match="bf16, f16 or f32"):
        shim.fp4_write_rows(rows.double(), rows.double(), slots, c.tensor, *geo, c.strides)
    with pytest.raises(RuntimeError, match="on the device"):
        shim.fp4_read_rows(c.tensor, *geo, 2, 64, c.strides, slots, torch.bfloat16)
    with pytest.raises(RuntimeError, match="bf16, f16 or f32"):
        shim.fp4_read_rows(c.tensor, *geo, 2, 64, c.strides, slots, torch.int8)
    q, tables, lens = torch.zeros(1, 4, 64).half(), torch.zeros(1, 2).int(), torch.ones(1).int()
    with pytest.raises(RuntimeError, match="on the"):
        shim.fp4_attend(q, c.tensor, *geo, 2, c.strides, tables, lens)
    with pytest.raises(RuntimeError, match="bf16 or f16"):
        shim.fp4_attend(q.float(), c.tensor, *geo, 2, c.strides, tables, lens)
    with pytest.raises(RuntimeError, match="must be on the device"):
        shim.copy_blocks(slots, slots.int(), slots.int(), 4, 2, 36, 16, c.strides, 1)
    with pytest.raises(RuntimeError, match="sources"):
        shim.copy_blocks(slots, slots.int(), slots[:2].int(), 4, 2, 36, 16, c.strides, 1)
    with pytest.raises(RuntimeError, match="on the\\s+device"):
        shim.plan_compaction(tables, None, 4)
    with pytest.raises(ValueError, match="expected"):
        c.write(slots, rows[:, :1], rows[:, :1])
    with pytest.raises(ValueError, match="expected"):
        c.attend(q[..., :32], tables, lens)
