"""Attention over full-width pages on the GPU against the oracle in 64 bits, behind shared prefixes and
without, and the weights that tokens get of it."""

import math

import numpy as np
import pytest
import torch

from everserve_amd.state.full import FullCache, SharedPrefix
from oracle import full

pytestmark = pytest.mark.gpu

LAYOUTS = ["kv_first", "blocks_first", "combined"]
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def shape_of(layout, blocks, bs, heads, d):
    return {"kv_first": (2, blocks, bs, heads, d), "blocks_first": (blocks, 2, bs, heads, d),
            "combined": (blocks, heads, bs, 2 * d)}[layout]


def canonical(cache):
    return full.canonical(cache.tensor.double().cpu().numpy(), cache.layout.value)


class Batch:
    """A cache whose rows hold no number but where a context's tokens are, sequences and prefixes
    with pages of their own in it, and queries that are views of a wider tensor."""

    def __init__(self, layout, bs, heads, shared, d, dtype, lens, news, seed=1, prefixes=(),
                 groups=(0,)):
        g = torch.Generator().manual_seed(seed)
        dtype = TYPES[dtype]
        every = list(prefixes) + list(lens)
        pages = [-(-n // bs) for n in every]
        blocks = sum(pages) + 3
        cache = torch.full(shape_of(layout, blocks, bs, heads, d), math.nan, dtype=dtype)
        perm = torch.randperm(blocks, generator=g).int()
        view = full.canonical(cache.view(torch.int16).numpy(), layout)
        tables = torch.full((len(every), max(1, max(pages, default=1)) + 1), 2 ** 30,
                            dtype=torch.int32)
        at = 0
        for i, n in enumerate(every):
            tables[i, :pages[i]] = perm[at:at + pages[i]]
            at += pages[i]
            if n:
                x = torch.randn(n, heads, 2, d, generator=g)
                x[:, :, 0] *= 1 + 3 * (torch.rand(d, generator=g) > 0.9)
                t = np.arange(n)
                view[tables[i].numpy()[t // bs], t % bs] = x.to(dtype).view(torch.int16).numpy()
        self.cache = FullCache(cache.cuda(), layout)
        self.lens, self.starts = list(lens), np.concatenate(([0], np.cumsum(news))).astype(int)
        self.tables, self.prefix_tables = tables[len(prefixes):], tables[:len(prefixes)]
        self.prefixes, self.groups, self.news = list(prefixes), list(groups), list(news)
        fused = torch.randn(int(self.starts[-1]), heads * shared + 2, d, generator=g).mul_(1.5)
        self.q = fused.to(dtype).cuda()[:, :heads * shared]
        self.mass = torch.rand(blocks, heads, bs, generator=g).pow(6).mul(9).cuda()

    def prefix(self, **how):
        if not self.prefixes:
            return None
        return SharedPrefix(self.prefix_tables.cuda(), ints(self.prefixes), ints(self.groups), **how)

    def attend(self, mass=None, scale=None, prefix_len=0, **how):
        if any(n != 1 for n in self.news):
            how = dict(q_starts=ints(self.starts.tolist()), max_q=max(self.news), **how)
        return self.cache.attend(self.q, self.tables.cuda(), ints(self.lens), scale=scale,
                                 return_lse=True, prefix=self.prefix(max_len=prefix_len),
                                 mass=mass, **how)

    def check(self, scale=None, **how):
        """Both calls of the batch, with mass and without, against the oracle."""
        out, lse = self.attend(scale=scale, **how)
        mass = self.mass.clone()
        again = self.attend(mass=mass, scale=scale, **how)
        assert torch.equal(again[0], out) and torch.equal(again[1], lse)
        prefix = (self.prefix_tables.numpy(), self.prefixes, self.groups) if self.prefixes else None
        want_mass = self.mass.double().cpu().numpy()
        d = self.q.shape[2]
        want = full.attend(self.q.double().cpu().numpy(), canonical(self.cache),
                           self.tables.numpy(), self.lens, self.starts, scale or d ** -0.5, prefix,
                           want_mass)
        compare(want, d, self.q.dtype, max(self.lens, default=0) + max(self.prefixes, default=0),
                out, lse)
        compare_mass(want, want_mass, d, self.q.shape[0] * self.q.shape[1] // self.cache.num_heads,
                     max(self.lens, default=0) + max(self.prefixes, default=0), mass)


def doubts(want, d, tokens):
    """How far a score, and a weight relative to itself, may be off.

    A score is a sum of d exact products in f32, in some order: off by at most
    (d + 4) 2^-24 sum |q_j k_j| scale, and by 2^-22 of itself from the scaling and the exponent's
    argument. A weight then is off by that, its exponential's 2^-22; the sums over n tokens and the
    joins add n 2^-24 of the weights' total."""
    worst = want["worst"]
    score = (d + 4) * 2.0 ** -24 * worst + 2.0 ** -22 * worst + 2.0 ** -22
    return score, 2 * score + 2 * (tokens + 16) * 2.0 ** -24


def compare(want, d, dtype, tokens, out, lse):
    """``out`` and ``lse`` against the oracle, within what the roundings may add up to: the weights'
    own (doubts) and theirs to the cache's type, half a step of it, or for f16 below 2^-14 half a
    step of 2^-24 beside a total of at least 1, and the output's rounding."""
    score, weight = doubts(want, d, tokens)
    half = HALF_STEP[dtype]
    room = want["reach"] * (weight[..., None] + half * (1 + weight[..., None]))
    least = 2.0 ** -25 if dtype == torch.float16 else 0.0
    room += least * want["values"]
    room += (np.abs(want["out"]) + room) * half + least + 1e-30
    off = np.abs(out.double().cpu().numpy() - want["out"])
    assert np.all(off <= room), float((off / room).max())
    got = lse.double().cpu().numpy()
    empty = np.isneginf(want["lse"])
    assert np.array_equal(np.isneginf(got), empty)
    off = np.abs(got[~empty] - want["lse"][~empty])
    room = (weight + 2.0 ** -21 * (1 + np.abs(np.where(empty, 0, want["lse"]))))[~empty]
    assert np.all(off <= room), float((off / room).max())


def compare_mass(want, mass, d, rows, tokens, got):
    """The masses: a weight exp(score - lse) is off by its score's doubt, the lse's and the
    exponential's, each relative to itself; the sum over the rows and the old mass add `rows` 2^-24
    of it."""
    per = (d + 4) * 2.0 ** -24 + 2.0 ** -22
    relative = want["doubt"] * (3 * per + 2.0 ** -20) + want["gave"] * (
        4 * (tokens + 16) * 2.0 ** -24 + 2.0 ** -20)
    room = relative + mass * (rows + 4) * 2.0 ** -24 + 1e-30
    off = np.abs(got.double().cpu().numpy() - mass)
    assert np.all(off <= room), float((off / room).max())


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("d", [16, 24, 32, 64, 72, 80, 96, 112, 120, 128, 136, 160, 192, 200, 256])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_single_tokens_over_every_head_size(ext, layout, d, dtype):
    Batch(layout, 16, 2, 3, d, dtype, [1, 77, 300, 0, 33], [1] * 5, seed=d).check()


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("d", [16, 64, 80, 104, 128, 136, 200, 256])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_single_tokens_behind_prefixes(ext, layout, d, dtype):
    Batch(layout, 16, 2, 3, d, dtype, [1, 77, 30, 0, 33, 5, 0], [1] * 7, seed=d,
          prefixes=[150, 37, 0], groups=[0, 3, 5, 7]).check()


@pytest.mark.parametrize("bs", [1, 3, 8, 16, 24, 64, 1000])
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 257, 513])
def test_contexts_that_end_anywhere_in_a_tile_or_a_page(ext, bs, n):
    Batch(LAYOUTS[n % 3], bs, 2, 2, 64, "bf16", [n, max(0, n - 1), n + 1], [1] * 3, seed=n,
          prefixes=[n + 1, n], groups=[0, 1, 3]).check()


@pytest.mark.parametrize("heads,shared", [(1, 1), (1, 8), (2, 7), (3, 16), (1, 17), (2, 40), (8, 4)])
@pytest.mark.parametrize("layout", LAYOUTS)
def test_heads_that_share(ext, heads, shared, layout):
    Batch(layout, 16, heads, shared, 128, "bf16", [65, 200], [1, 1], seed=heads).check()
    Batch(layout, 16, heads, shared, 128, "bf16", [65, 20, 1], [1] * 3, seed=heads, prefixes=[99],
          groups=[0, 3]).check()


@pytest.mark.parametrize("d", [64, 80, 128, 192])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("bs", [16, 24])
def test_chunks_of_queries_see_what_is_before_them(ext, d, dtype, bs):
    # a whole prompt, a chunk after more, single tokens, more queries than tokens (rows that see
    # nothing), an empty context with queries, a sequence without queries
    lens, news = [70, 150, 33, 5, 0, 40, 1, 260], [70, 37, 1, 9, 3, 0, 1, 130]
    Batch(LAYOUTS[d % 3], bs, 2, 4, d, dtype, lens, news, seed=d).check()
    Batch(LAYOUTS[d % 3], bs, 2, 4, d, dtype, lens, news, seed=d, prefixes=[100, 20],
          groups=[1, 4, 7]).check()


@pytest.mark.parametrize("shared", [1, 5, 32])
@pytest.mark.parametrize("news", [[2, 3, 1], [17, 1, 64], [150, 129, 97]])
def test_few_and_many_queries_of_a_sequence(ext, shared, news):
    Batch("combined", 32, 1, shared, 64, "bf16", [200, 131, 100], news, seed=shared).check()
    Batch("combined", 32, 1, shared, 64, "bf16", [160, 131, 100], news, seed=shared,
          prefixes=[90], groups=[0, 2]).check()


@pytest.mark.parametrize("lens", [[4097], [9000, 3], [2500] * 3])
@pytest.mark.parametrize("news", [1, 4])
@pytest.mark.parametrize("before", [0, 5000])
def test_long_contexts_are_split_and_joined(ext, lens, news, before):
    Batch("combined", 16, 1, 4, 128, "bf16", lens, [news] * len(lens), seed=news,
          prefixes=[before] if before else [], groups=[0, len(lens)]).check()


@pytest.mark.parametrize("max_len", [1, 17, 300, 10 ** 9])
def test_bounds_on_lengths_only_steer(ext, max_len):
    b = Batch("kv_first", 16, 2, 4, 64, "bf16", [700, 3, 1500], [1, 1, 1], prefixes=[900],
              groups=[1, 3])
    b.check(max_len=max_len, prefix_len=max_len)
    b = Batch("kv_first", 16, 2, 4, 64, "bf16", [700, 30, 90], [40, 1, 90], prefixes=[900],
              groups=[1, 3])
    b.check(max_len=max_len, prefix_len=max_len)


def test_a_peaked_row_and_large_scores(ext):
    Batch("kv_first", 16, 2, 4, 64, "bf16", [500, 90], [1, 1], prefixes=[70], groups=[0, 1]).check(
        scale=3.0)
    Batch("kv_first", 16, 2, 4, 64, "f16", [500, 90], [40, 1]).check(scale=0.001)


def test_sequences_in_no_group(ext):
    Batch("kv_first", 16, 2, 2, 64, "bf16", [40, 3, 17, 0, 60], [1] * 5, prefixes=[70, 33],
          groups=[1, 2, 4]).check()
    Batch("kv_first", 16, 2, 2, 64, "bf16", [40, 9, 17, 0, 60], [5, 3, 1, 2, 20],
          prefixes=[70, 33, 5], groups=[1, 2, 2, 4]).check()


@pytest.mark.parametrize("seqs", [257, 600])
def test_more_sequences_and_groups_than_a_workgroup_has_threads(ext, seqs):
    lens = [(37 * i) % 40 for i in range(seqs)]
    lens[seqs // 2], lens[-1] = 500, 310
    for news in ([1] * seqs, [1 + (i % 3) * 9 for i in range(seqs)]):
        Batch("kv_first", 16, 1, 2, 16, "bf16", lens, news, seed=seqs,
              prefixes=[5 + i % 30 for i in range(seqs // 2)],
              groups=list(range(0, 2 * (seqs // 2) + 1, 2))).check()


@pytest.mark.parametrize("news", [1, 40])
def test_pages_that_the_cache_does_not_have_hold_nothing(ext, news):
    for d, bs in ((64, 16), (128, 24)):
        b = Batch("kv_first", bs, 2, 2, d, "bf16", [400, 130, 90], [news] * 3, seed=4,
                  prefixes=[200, 50], groups=[0, 2, 3])
        b.tables[0, 3], b.tables[0, 5], b.tables[0, 6] = -1, b.cache.num_blocks, -(2 ** 31)
        b.tables[1, 0] = 2 ** 31 - 1
        b.tables[2, :] = -5
        b.prefix_tables[0, 2], b.prefix_tables[1, :] = -1, 2 ** 30
        b.check()
        out, lse = b.attend()
        assert torch.all(out[2 * news:] == 0) and torch.all(lse[2 * news:] == -math.inf)


def test_lengths_and_starts_past_their_arrays_are_cut(ext):
    b = Batch("combined", 16, 1, 2, 64, "bf16", [64, 64], [2, 2], seed=5, prefixes=[32],
              groups=[0, 2])
    tables, q = b.tables[:, :4].contiguous().cuda(), b.q
    call = b.cache.attend
    out = call(q[:2], tables, ints([10 ** 9, -7]))
    assert torch.equal(out, call(q[:2], tables, ints([64, 0]))) and torch.all(out[1] == 0)
    out = call(q, tables, ints([64, 64]), q_starts=ints([-3, 2, 900]), max_q=4)
    assert torch.equal(out, call(q, tables, ints([64, 64]), q_starts=ints([0, 2, 4]), max_q=2))
    pt = b.prefix_tables[:, :2].contiguous().cuda()
    want = call(q, tables, ints([64, 64]), q_starts=ints([0, 2, 4]), max_q=2,
                prefix=SharedPrefix(pt, ints([32]), ints([0, 2])))
    for pl, gs in (([10 ** 9], [0, 2]), ([32], [-5, 2]), ([32], [0, 77])):
        got = call(q, tables, ints([64, 64]), q_starts=ints([0, 2, 4]), max_q=2,
                   prefix=SharedPrefix(pt, ints(pl), ints(gs)))
        assert torch.equal(got, want), (pl, gs)
    none = call(q, tables, ints([64, 64]), q_starts=ints([0, 2, 4]), max_q=2)
    for pl, gs in (([-3], [0, 2]), ([32], [2, 2]), ([32], [2, 0])):
        got = call(q, tables, ints([64, 64]), q_starts=ints([0, 2, 4]), max_q=2,
                   prefix=SharedPrefix(pt, ints(pl), ints(gs)))
        assert torch.equal(got, none), (pl, gs)


@pytest.mark.parametrize("d,dtype", [(64, "bf16"), (80, "f16"), (128, "bf16"), (256, "f16")])
@pytest.mark.parametrize("news,shared", [(3, 4), (16, 1), (100, 2), (33, 5)])
@pytest.mark.parametrize("back", [0, 1, 2, 40])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_no_number_in_a_masked_place(ext, d, dtype, news, shared, back, bad):
    """A token whose V holds no finite number, among the last places of a chunk: the rows before it
    are as without it, in the same products' tile."""
    n = 200
    b = Batch("kv_first", 16, 1, shared, d, dtype, [n, n], [news] * 2, seed=6)
    at = n - 1 - back
    row = b.cache.tensor[:, int(b.tables[0, at // 16]), at % 16, 0]  # K, V
    row[1, d - 10] = 1
    want, _ = b.attend()
    row[1, d - 10] = bad
    out, _ = b.attend()
    hit = max(news - 1 - back, 0)  # the first query that sees the token
    wild = ~torch.isfinite(out)
    assert wild[hit:news, :, d - 10].all()
    wild[hit:news, :, d - 10] = False
    assert not wild.any()
    same = torch.ones_like(wild)
    same[hit:news, :, d - 10] = False
    assert torch.equal(out[same], want[same])
    if bad == math.inf:
        assert torch.all(out[hit:news, :, d - 10] == math.inf)
    # and a K without a number: the rows that see it are none, the others as they were
    row[0, d - 10], row[1, d - 10] = math.nan, 1
    out, _ = b.attend()
    assert torch.isnan(out[hit:news]).all() and torch.equal(out[:hit], want[:hit])
    assert torch.equal(out[news:], want[news:])


def test_padding_queries_that_no_sequence_names_are_left_alone(ext):
    b = Batch("kv_first", 16, 1, 4, 64, "bf16", [300, 40], [45, 45], seed=6, prefixes=[100],
              groups=[0, 2])
    lens, tables = ints([300, 40]), b.tables.cuda()
    for starts in ([0, 1, 31], [3, 60, 62], [10, 10, 50]):
        out = torch.full_like(b.q, 7.0, memory_format=torch.contiguous_format)
        mass, own_mass = b.mass.clone(), b.mass.clone()
        b.cache.attend(b.q, tables, lens, q_starts=ints(starts), max_q=60, out=out,
                       prefix=b.prefix(), mass=mass)
        assert torch.all(out[:starts[0]] == 7) and torch.all(out[starts[2]:] == 7)
        part = b.q[starts[0]:starts[2]].contiguous()
        want = b.cache.attend(part, tables, lens, q_starts=ints([s - starts[0] for s in starts]),
                              max_q=60, prefix=b.prefix(), mass=own_mass)
        assert torch.equal(out[starts[0]:starts[2]], want)
        assert torch.equal(mass, own_mass)


def test_queries_past_max_q_are_left_alone_and_weigh_nothing(ext):
    b = Batch("kv_first", 16, 1, 4, 64, "bf16", [300, 40], [45, 45], seed=6, prefixes=[100],
              groups=[0, 2])
    lens, tables, starts = ints([300, 40]), b.tables.cuda(), ints([0, 45, 90])
    out = torch.full_like(b.q, 7.0, memory_format=torch.contiguous_format)
    mass, own_mass = b.mass.clone(), b.mass.clone()
    b.cache.attend(b.q, tables, lens, q_starts=starts, max_q=20, out=out, prefix=b.prefix(),
                   mass=mass)
    kept = torch.cat((torch.arange(20), torch.arange(45, 65))).cuda()
    want = b.cache.attend(b.q[kept].contiguous(), tables, lens, q_starts=ints([0, 20, 40]),
                          max_q=20, prefix=b.prefix(), mass=own_mass)
    assert torch.equal(out[kept], want)
    assert torch.all(out[20:45] == 7) and torch.all(out[65:] == 7)
    # the rows lie in other tiles of 16: the same weights in another order of sums
    assert torch.allclose(mass, own_mass, rtol=1e-5, atol=0)


@pytest.mark.parametrize("how", ["no sequence", "no query"])
def test_rows_without_work_are_zeros(ext, how):
    b = Batch("kv_first", 16, 2, 4, 64, "bf16", [40, 7], [3, 4], prefixes=[9], groups=[0, 2])
    tables, lens, starts, max_q, prefix = b.tables.cuda(), ints(b.lens), ints([0, 0, 0]), 5, None
    if how == "no query":
        max_q, prefix = 0, b.prefix()
    else:
        tables, lens, starts = tables[:0], lens[:0], starts[:1]
    for _ in range(3):
        held = [torch.full((7, 4, 64), math.nan, device="cuda") for _ in range(3)]
        torch.cuda.synchronize()
        del held
        mass = b.mass.clone()
        out, lse = b.cache.attend(b.q, tables, lens, q_starts=starts, max_q=max_q, return_lse=True,
                                  prefix=prefix, mass=mass)
        assert torch.all(out == 0) and torch.all(lse == -math.inf) and torch.equal(mass, b.mass)


def test_views_of_wider_tensors(ext):
    """A head slice of a cache, tables that are views, queries whose tokens lie apart."""
    b = Batch("blocks_first", 16, 4, 2, 72, "bf16", [150, 33, 70], [1, 3, 9], seed=3,
              prefixes=[60], groups=[0, 2])
    part = FullCache(b.cache.tensor[:, :, :, 1:3], "blocks_first")
    apart = torch.full((5, b.tables.shape[1] + 7), -9, dtype=torch.int32)
    apart[1:4, 2:2 + b.tables.shape[1]] = b.tables
    view = apart.cuda()[1:4, 2:2 + b.tables.shape[1]]
    starts = ints(b.starts.tolist())
    whole, _ = b.attend()
    out = part.attend(b.q[:, 2:6], view, ints(b.lens), q_starts=starts, max_q=9, prefix=b.prefix())
    assert torch.equal(out, whole[:, 2:6])
    one = view[:1].expand(3, -1)  # three sequences of one table
    out = b.cache.attend(b.q[:3], one, ints([150, 17, 0]))
    want = b.cache.attend(b.q[:3], one.contiguous(), ints([150, 17, 0]))
    assert torch.equal(out, want) and torch.all(out[2] == 0)


def test_pages_past_four_gigabytes(ext):
    # 2^32 bytes lie between the first page and the last
    heads, d, bs = 8, 256, 64
    blocks = (1 << 32) // (heads * bs * 2 * 2 * d) + 9
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(3, heads, bs, 2 * d, device="cuda", generator=g).bfloat16()
    q = torch.randn(1, 16, d, device="cuda", generator=g).bfloat16()
    outs = []
    for n, pages in ((blocks, [blocks - 1, 0, blocks - 2]), (3, [0, 1, 2])):
        t = torch.empty(n, heads, bs, 2 * d, dtype=torch.bfloat16, device="cuda")
        t[torch.tensor(pages, device="cuda")] = x
        mass = torch.zeros(n, heads, bs, device="cuda")
        out = FullCache(t, "combined").attend(q, ints([pages[1:]]), ints([100]), mass=mass,
                                              prefix=SharedPrefix(ints([pages[:1]]), ints([50]),
                                                                  ints([0, 1])))
        outs.append((out, mass[torch.tensor(pages, device="cuda")]))
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])


def test_the_same_call_gives_the_same_bits_and_out_is_written_in_place(ext):
    b = Batch("combined", 16, 2, 4, 128, "bf16", [5000, 900, 77], [1] * 3, seed=8, prefixes=[3001],
              groups=[0, 3])
    out = torch.full_like(b.q, 3.0, memory_format=torch.contiguous_format)
    mass = b.mass.clone()
    assert b.attend(out=out, mass=mass)[0] is out
    for _ in range(3):
        again = b.mass.clone()
        assert torch.equal(b.attend(mass=again)[0], out) and torch.equal(again, mass)


def test_mass_of_several_steps_adds_up(ext):
    b = Batch("kv_first", 16, 2, 2, 64, "bf16", [50, 20], [1, 1], seed=2, prefixes=[40],
              groups=[0, 2])
    mass, one = torch.zeros_like(b.mass), torch.zeros_like(b.mass)
    for _ in range(3):
        b.attend(mass=mass)
    b.attend(mass=one)
    fresh = torch.zeros_like(one, dtype=torch.bool)  # the newest tokens start afresh every time
    for s, n in enumerate(b.lens):
        fresh[int(b.tables[s, (n - 1) // 16]), :, (n - 1) % 16] = True
    assert torch.equal(mass[fresh], one[fresh])
    assert torch.allclose(mass[~fresh], 3 * one[~fresh], rtol=2.0 ** -22, atol=0)
    # what a step gives is one of each row
    assert abs(float(one.double().sum()) - 2 * 4) < 1e-4


def test_the_calls_run_on_their_stream_behind_its_work(ext):
    b = Batch("kv_first", 16, 2, 4, 128, "bf16", [3000, 200, 77], [1, 40, 3], seed=8,
              prefixes=[900], groups=[0, 2])
    tables, prefix, starts = b.tables.cuda(), b.prefix(), ints(b.starts.tolist())
    a = torch.randn(8192, 8192, device="cuda", dtype=torch.bfloat16)
    c = torch.empty_like(a)
    q, lens = torch.zeros_like(b.q, memory_format=torch.contiguous_format), ints([1, 1, 1])
    masses = [b.mass.clone(), b.mass.clone()]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    how = dict(q_starts=starts, max_q=40, return_lse=True, prefix=prefix)
    with torch.cuda.stream(side):
        for _ in range(8):
            torch.mm(a, a, out=c)
        q.copy_(b.q)
        lens.copy_(ints(b.lens))
        got = b.cache.attend(q, tables, lens, mass=masses[0], **how)
    side.synchronize()
    want = b.cache.attend(b.q, tables, ints(b.lens), mass=masses[1], **how)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(masses[0], masses[1])


def test_a_captured_batch_replays_with_other_lengths(ext):
    b = Batch("combined", 16, 2, 4, 64, "bf16", [4000, 900, 900, 900], [81, 3, 3, 3], seed=8,
              prefixes=[700, 300], groups=[0, 2, 4])
    dev, lens = b.tables.cuda(), ints([3000, 40, 700, 0])
    starts, pl, gs = ints([0, 1, 2, 80, 81]), ints([700, 300]), ints([0, 2, 4])
    prefix = SharedPrefix(b.prefix_tables.cuda(), pl, gs)

    def step(mass):
        return b.cache.attend(b.q, dev, lens, q_starts=starts, max_q=80, return_lse=True,
                              prefix=prefix, mass=mass)

    masses = [b.mass.clone(), b.mass.clone()]
    step(masses[0])
    masses[0].copy_(b.mass)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(masses[0])
    for new, at, before, members in (
            ([3000, 40, 700, 0], [0, 1, 2, 80, 81], [700, 300], [0, 2, 4]),
            ([4000, 900, 80, 3], [0, 9, 10, 11, 90], [1, 0], [0, 1, 4]),
            ([1, 2, 3, 4], [0, 1, 2, 3, 4], [650, 299], [1, 1, 3]),
            ([0, 0, 900, 900], [0, 80, 81, 82, 90], [0, 5], [0, 4, 4])):
        for x, y in ((lens, new), (starts, at), (pl, before), (gs, members)):
            x.copy_(torch.tensor(y, dtype=torch.int32))
        graph.replay()
        want = step(masses[1])
        torch.cuda.synchronize()
        n = at[-1]
        assert torch.equal(got[0][:n], want[0][:n]) and torch.equal(got[1][:n], want[1][:n])
        assert torch.equal(masses[0], masses[1])


def test_calls_on_two_streams_at_once(ext):
    b = Batch("kv_first", 16, 2, 4, 128, "bf16", [3000, 200, 77], [1] * 3, seed=8, prefixes=[900],
              groups=[0, 2])
    want = b.attend()
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(b.attend())
    torch.cuda.synchronize()
    assert all(torch.equal(a[0], want[0]) and torch.equal(a[1], want[1]) for a in got)


def test_what_it_cannot_do_is_refused(ext):
    b = Batch("combined", 16, 1, 2, 64, "bf16", [10, 5], [1, 1], seed=8, prefixes=[7],
              groups=[0, 2])
    call, q = b.cache.attend, b.q.contiguous()
    tables, lens = b.tables.cuda(), ints([10, 5])
    with pytest.raises(RuntimeError, match="backward"):
        call(q.clone().requires_grad_(), tables, lens)
    with torch.no_grad():
        assert torch.isfinite(call(q.clone().requires_grad_(), tables, lens)).all()
    with pytest.raises(RuntimeError, match="lengths"):
        call(q, tables, lens[:1])
    with pytest.raises(RuntimeError, match="query starts"):
        call(q, tables, lens, q_starts=lens)
    with pytest.raises(RuntimeError, match="out must"):
        call(q, tables, lens, out=torch.zeros(2, 2, 64, device="cuda"))
    with pytest.raises(RuntimeError, match="int32"):
        call(q, tables.long(), lens)
    with pytest.raises(RuntimeError, match="cache's type"):
        call(q.half(), tables, lens)
    with pytest.raises(RuntimeError, match="16 bytes"):
        call(torch.zeros(2, 2, 72, device="cuda").bfloat16()[..., 1:65], tables, lens)
    with pytest.raises(RuntimeError, match="mass of shape"):
        call(q, tables, lens, mass=b.mass[:-1])
    with pytest.raises(RuntimeError, match="mass must be"):
        call(q, tables, lens, mass=b.mass.double())
    for bad in (SharedPrefix(b.prefix_tables.cuda(), ints([7, 7]), ints([0, 2])),
                SharedPrefix(b.prefix_tables.cuda(), ints([7]), ints([0, 1, 2]))):
        with pytest.raises(RuntimeError, match="prefixes"):
            call(q, tables, lens, prefix=bad)
    with pytest.raises(RuntimeError, match="scale"):
        call(q, tables, lens, scale=-1.0)


def test_an_output_that_is_the_queries_is_refused(ext):
    b = Batch("kv_first", 16, 2, 2, 64, "bf16", [20, 33], [1] * 2)
    b.q = b.q.contiguous()
    with pytest.raises(RuntimeError, match="must not be the queries"):
        b.attend(out=b.q)


@pytest.mark.parametrize("queries", [5, 16])
@pytest.mark.parametrize("seqs", [8, 30, 60])
def test_small_chunks_behind_a_prefix_on_both_sides_of_the_wide_tiles(ext, seqs, queries):
    lens = [(7 * s + queries) % 61 + queries for s in range(seqs)]
    Batch("kv_first", 16, 1, 4, 64, "bf16", lens, [queries] * seqs, seed=seqs, prefixes=[300],
          groups=[0, seqs]).check()


@pytest.mark.parametrize("n", [1023, 1024, 1025])
def test_contexts_that_are_just_one_part_and_just_two(ext, n):
    Batch("combined", 16, 2, 4, 64, "bf16", [n, 5, n - 700], [1] * 3, seed=n).check(max_len=n)
