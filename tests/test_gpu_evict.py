"""Eviction on the GPU against the oracle: the tokens that stay, and every byte of the caches and
masses after it."""

import math

import numpy as np
import pytest
import torch

from everserve_amd.state.evict import Evictor
from everserve_amd.state.fp4 import row_bytes
from oracle import full

pytestmark = pytest.mark.gpu

LAYOUTS = ["kv_first", "blocks_first", "combined"]
TYPES = {"bf16": (torch.int16, torch.bfloat16), "f32": (torch.int32, torch.float32),
         "fp8": (torch.uint8, torch.uint8)}


def ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def shape_of(layout, blocks, bs, heads, d):
    return {"kv_first": (2, blocks, bs, heads, d), "blocks_first": (blocks, 2, bs, heads, d),
            "combined": (blocks, heads, bs, 2 * d)}[layout]


def masses(shape, g, kind):
    x = torch.rand(shape, generator=g)
    if kind == "ties":
        return torch.floor(x * 4) / 4
    if kind == "wild":
        x = torch.where(x < 0.3, -x, x) * 10.0 ** torch.randint(-30, 30, shape, generator=g)
        for v, p in ((math.nan, 0.05), (-math.nan, 0.03), (math.inf, 0.05), (-math.inf, 0.05),
                     (0.0, 0.1), (-0.0, 0.1)):
            x[torch.rand(shape, generator=g) < p] = v
        return x
    return x.pow(8) * 50


class Case:
    def __init__(self, layout, dtype, layers, heads, d, bs, lens, budget, recent, kind="plain",
                 seed=1):
        g = torch.Generator().manual_seed(seed)
        pages = [-(-n // bs) for n in lens]
        room = -(-budget // bs)
        blocks = sum(pages) + len(lens) * room + 2
        store, dt = TYPES[dtype]
        info = torch.iinfo(store)
        self.tensors = [torch.randint(info.min, info.max, shape_of(layout, blocks, bs, heads, d),
                                      dtype=store, generator=g).cuda() for _ in range(layers)]
        perm = torch.randperm(blocks, generator=g).int()
        self.tables = torch.full((len(lens), max(1, max(pages))), 2 ** 30, dtype=torch.int32)
        self.new = torch.zeros((len(lens), max(1, room)), dtype=torch.int32)
        at = 0
        for s in range(len(lens)):
            self.tables[s, :pages[s]] = perm[at:at + pages[s]]
            at += pages[s]
            self.new[s, :room] = perm[at:at + room]
            at += room
        self.lens, self.budget, self.recent, self.layout = lens, budget, recent, layout
        self.mass = masses((layers, blocks, heads, bs), g, kind).cuda()
        self.evictor = Evictor([t.view(dt) for t in self.tensors], layout)

    def check(self):
        want = [full.canonical(t.cpu().numpy().copy(), self.layout) for t in self.tensors]
        mass = self.mass.cpu().numpy().copy()
        lens, kept = full.evict(want, mass, self.tables.numpy(), self.lens, self.new.numpy(),
                                self.budget, self.recent)
        got = self.evictor.evict(self.tables.cuda(), ints(self.lens), self.new.cuda(), self.budget,
                                 self.mass, recent=self.recent)
        assert np.array_equal(got.lens.cpu().numpy(), lens)
        assert np.array_equal(got.kept.cpu().numpy(), kept)
        for t, w in zip(self.tensors, want):
            assert np.array_equal(full.canonical(t.cpu().numpy(), self.layout), w)
        assert np.array_equal(self.mass.cpu().numpy().view(np.int32), mass.view(np.int32))


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("d", [16, 36, 64, 120, 128])
def test_rows_of_every_kind(ext, layout, dtype, d):
    Case(layout, dtype, 2, 3, d, 16, [70, 33, 0, 1, 200, 40], 40, 9, seed=d).check()


@pytest.mark.parametrize("kind", ["plain", "ties", "wild"])
@pytest.mark.parametrize("budget,recent", [(1, 0), (1, 1), (7, 7), (64, 0), (100, 33), (500, 100),
                                           (1000, 999)])
@pytest.mark.parametrize("bs", [1, 16, 24])
def test_budgets_and_orders(ext, kind, budget, recent, bs):
    lens = [budget - 1, budget, budget + 1, 3 * budget, 777]
    Case("kv_first", "bf16", 1, 2, 16, bs, lens, budget, recent, kind, seed=budget).check()


@pytest.mark.parametrize("n", [511, 512, 513, 4095, 4096, 4097, 8191, 8193, 12289, 20000, 70001])
@pytest.mark.parametrize("kind", ["plain", "ties"])
def test_long_contexts(ext, n, kind):
    Case("combined", "fp8", 1, 1, 16, 64, [n, n // 2], n // 3, n // 30, kind, seed=n).check()


def test_all_masses_alike_and_none(ext):
    for value in (0.0, 1.0, math.nan, -math.inf):
        c = Case("kv_first", "bf16", 1, 2, 16, 16, [9000, 300], 200, 10)
        c.mass.fill_(value)
        c.check()


def test_a_four_bit_caches_rows(ext):
    Case("combined", "fp8", 3, 3, row_bytes(96), 24, [300, 0, 71], 50, 7).check()
    Case("kv_first", "fp8", 2, 5, row_bytes(80), 16, [300, 0, 71], 50, 7).check()


def test_many_heads_and_one_long_row(ext):
    Case("kv_first", "bf16", 1, 70, 16, 16, [90, 40], 33, 3).check()
    Case("blocks_first", "f32", 1, 1, 1000, 16, [90, 40], 33, 3).check()


def test_pages_that_the_cache_does_not_have(ext):
    c = Case("kv_first", "bf16", 2, 2, 32, 16, [200, 150, 90], 64, 20)
    c.tables[0, 3], c.tables[0, 11], c.tables[1, :] = -1, 2 ** 30, -7
    c.new[0, 1], c.new[2, 3] = 2 ** 31 - 1, -1
    c.check()


def test_pages_that_others_share_are_left_as_they_are(ext):
    c = Case("kv_first", "bf16", 2, 2, 32, 16, [200, 200], 64, 20)
    c.tables[1] = c.tables[0]  # both sequences of one context
    before = [t.clone() for t in c.tensors]
    c.check()
    pages = c.tables[0].long().cuda()
    for t, b in zip(c.tensors, before):
        assert torch.equal(t[:, pages], b[:, pages])


def test_lengths_past_their_tables_and_tables_that_are_views(ext):
    c = Case("kv_first", "bf16", 1, 2, 32, 16, [160, 48, 0], 64, 20)
    c.lens = [10 ** 9, 48, -3]
    apart = torch.full((3, 40), -9, dtype=torch.int32)
    apart[:, 5:5 + c.tables.shape[1]] = c.tables
    view = apart.cuda()[:, 5:5 + c.tables.shape[1]]
    want = [full.canonical(t.cpu().numpy().copy(), "kv_first") for t in c.tensors]
    lens, kept = full.evict(want, c.mass.cpu().numpy().copy(), c.tables.numpy(), c.lens,
                            c.new.numpy(), 64, 20)
    got = c.evictor.evict(view, ints(c.lens), c.new.cuda(), 64, c.mass, recent=20)
    assert np.array_equal(got.lens.cpu().numpy(), lens)
    assert np.array_equal(got.kept.cpu().numpy(), kept)
    assert np.array_equal(full.canonical(c.tensors[0].cpu().numpy(), "kv_first"), want[0])


def test_nothing_to_keep_and_no_sequence(ext):
    c = Case("kv_first", "bf16", 1, 2, 32, 16, [160, 0], 16, 0)
    before = c.tensors[0].clone()
    got = c.evictor.evict(c.tables.cuda(), ints(c.lens), c.new.cuda()[:, :0], 0, c.mass)
    assert got.lens.tolist() == [0, 0] and got.kept.shape == (1, 2, 2, 0)
    got = c.evictor.evict(c.tables.cuda()[:0], ints([]), c.new.cuda()[:0], 16, c.mass)
    assert got.lens.numel() == 0 and torch.equal(c.tensors[0], before)


def test_a_page_past_four_gigabytes(ext):
    heads, d, bs = 8, 256, 64
    blocks = (1 << 32) // (heads * bs * 2 * 2 * d) + 9
    t = torch.empty(blocks, heads, bs, 2 * d, dtype=torch.bfloat16, device="cuda")
    mass = torch.zeros(1, blocks, heads, bs, device="cuda")
    x = torch.randn(heads, bs, 2 * d, device="cuda").bfloat16()
    t[blocks - 1] = x
    mass[0, blocks - 1] = torch.arange(bs, device="cuda").float()
    got = Evictor([t], "combined").evict(ints([[blocks - 1]]), ints([bs]), ints([[0]]), 40, mass)
    assert torch.equal(t[0, :, :40], x[:, -40:]) and got.lens.tolist() == [40]
    got = Evictor([t], "combined").evict(ints([[0]]), ints([40]), ints([[blocks - 2]]), 40, mass)
    assert torch.equal(t[blocks - 2, :, :40], x[:, -40:])


def test_on_a_stream_and_in_a_graph(ext):
    cases = [Case("kv_first", "bf16", 2, 2, 64, 16, [900, 300, 50], 100, 11) for _ in range(2)]
    dev = [(c.tables.cuda(), ints(c.lens), c.new.cuda()) for c in cases]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def step(c, d):
        return c.evictor.evict(*d, c.budget, c.mass, recent=c.recent)

    with torch.cuda.stream(side):
        step(cases[0], dev[0])
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(cases[0], dev[0])
    g = torch.Generator(device="cuda").manual_seed(4)
    for lens in ([900, 300, 50], [90, 100, 56], [0, 101, 1]):
        mass = torch.rand(cases[0].mass.shape, device="cuda", generator=g)
        for c, d in zip(cases, dev):
            c.mass.copy_(mass)
            d[1].copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        want = step(cases[1], dev[1])
        torch.cuda.synchronize()
        assert torch.equal(got.lens, want.lens) and torch.equal(got.kept, want.kept)
        assert torch.equal(cases[0].mass, cases[1].mass)
        for a, b in zip(cases[0].tensors, cases[1].tensors):
            assert torch.equal(a, b)


def test_what_it_cannot_do_is_refused(ext):
    c = Case("kv_first", "bf16", 1, 2, 32, 16, [60, 40], 32, 4)
    tables, lens, new = c.tables.cuda(), ints(c.lens), c.new.cuda()
    call = c.evictor.evict
    with pytest.raises(RuntimeError, match="newest"):
        call(tables, lens, new, 32, c.mass, recent=33)
    with pytest.raises(RuntimeError, match="newest"):
        call(tables, lens, new, -1, c.mass)
    with pytest.raises(RuntimeError, match="hold no"):
        call(tables, lens, new, 33, c.mass)
    with pytest.raises(RuntimeError, match="lengths"):
        call(tables, lens[:1], new, 32, c.mass)
    with pytest.raises(RuntimeError, match="mass of shape"):
        call(tables, lens, new, 32, c.mass[0])
    with pytest.raises(RuntimeError, match="mass must be"):
        call(tables, lens, new, 32, c.mass.half())
    with pytest.raises(RuntimeError, match="int32"):
        call(tables.long(), lens, new, 32, c.mass)
    with pytest.raises(RuntimeError, match="on the\\s+device"):
        call(tables, lens, new.cpu(), 32, c.mass)
    with pytest.raises(ValueError, match="contiguous"):
        Evictor([torch.zeros(4, 2, 16, 2, 64, device="cuda")[..., ::2]], "blocks_first")
