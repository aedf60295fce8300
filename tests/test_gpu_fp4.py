"""The 4-bit cache on the GPU against the oracle in 64 bits: rows written and read, and attention."""

import math

import numpy as np
import pytest
import torch

from everserve_amd.state.fp4 import Fp4Cache, cache_shape
from oracle import fp4

pytestmark = pytest.mark.gpu

LAYOUTS = ["kv_first", "blocks_first", "combined"]
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def canonical(cache):
    return fp4.canonical(cache.tensor.cpu().numpy(), cache.layout.value)


def values(shape, seed, dtype):
    """Rows with groups of very different size, zeros, ties and the grid's own values."""
    g = np.random.default_rng(seed)
    x = g.standard_normal(shape) * np.exp2(g.integers(-12, 12, shape[:-1] + (1,)))
    x[g.random(shape) < 0.05] = 0
    flat = x.reshape(-1, shape[-1])
    ties = np.array([6, .25, .75, 1.25, 1.75, 2.5, 3.5, 5, -.25, -.75, -2.5, -5, 7, -0.0, 0, 1])
    flat[0, :16] = ties[:flat.shape[1]]
    flat[-1] = 0
    return torch.from_numpy(x).to(dtype)


# ---------------------------------------------------------------- rows
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("d", [16, 40, 64, 80, 96, 120, 128, 192, 256])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_rows_are_held_as_the_oracle_rounds_them(ext, layout, d, dtype):
    dtype, n, heads, bs = TYPES[dtype], 21, 3, 5
    cache = Fp4Cache(torch.full(cache_shape(layout, 7, bs, heads, d), 77, dtype=torch.uint8,
                                device="cuda"), d, layout)
    want = canonical(cache).copy()
    key, value = values((n, heads, d), d, dtype), values((n, heads, d), d + 1, dtype)
    slots = torch.randperm(35, generator=torch.Generator().manual_seed(d))[:n]
    slots[3], slots[9], slots[10] = -1, 35, -(2 ** 40)  # no slots of this cache
    # views of one fused tensor: rows are not contiguous with each other
    fused = torch.cat((key, value), 1).cuda()
    cache.write(slots.cuda(), fused[:, :heads], fused[:, heads:])
    for i, s in enumerate(slots.tolist()):
        if 0 <= s < 35:
            want[s // bs, s % bs, :, 0] = fp4.encode(key[i].double().numpy())
            want[s // bs, s % bs, :, 1] = fp4.encode(value[i].double().numpy())
    assert np.array_equal(canonical(cache), want)
    # back at full width, from rows of any bytes (a scale byte 77 among them)
    back = torch.tensor([0, -1, 34, 35, 7, 7, 2 ** 33] + list(range(35)))
    for t in TYPES.values():
        got = cache.read(back.cuda(), t)
        for kv in (0, 1):
            rows = np.zeros((len(back), heads, d))
            for i, s in enumerate(back.tolist()):
                if 0 <= s < 35:
                    rows[i] = fp4.decode(want[s // bs, s % bs, :, kv], d)
            assert got[kv].dtype == t and got[kv].shape == (len(back), heads, d)
            assert torch.equal(got[kv].cpu(), torch.from_numpy(rows).to(t))


@pytest.mark.parametrize("dtype", list(TYPES))
def test_groups_without_a_number_read_as_nan_and_extremes_hold(ext, dtype):
    dtype = TYPES[dtype]
    x = torch.ones(4, 2, 72, dtype=dtype)
    x[0, 0, 3], x[0, 1, 40], x[1, 0, 71] = math.nan, math.inf, -math.inf
    x[2] = torch.finfo(dtype).max
    x[3] = torch.finfo(dtype).tiny
    cache = Fp4Cache.empty(2, 3, 2, 72)
    slots = torch.arange(4, device="cuda")
    cache.write(slots, x.cuda(), -x.cuda())
    want = fp4.encode(x.double().numpy())
    assert np.array_equal(canonical(cache).reshape(6, 2, 2, -1)[:4, :, 0], want)
    key, value = cache.read(slots, torch.float32)
    assert torch.equal(torch.isnan(key.cpu()), torch.isnan(torch.from_numpy(fp4.decode(want, 72))))
    assert torch.equal(torch.nan_to_num(key), torch.nan_to_num(-value))


def test_rows_off_16_bytes_and_empty_lists(ext):
    heads, d, n = 2, 64, 9
    x = values((n, 2 * heads, d + 1), 3, torch.bfloat16).cuda()[..., 1:]  # rows on 2 bytes
    cache = Fp4Cache.empty(3, 4, heads, d, "kv_first")
    slots = torch.arange(n, device="cuda")
    cache.write(slots, x[:, :heads], x[:, heads:])
    got = canonical(cache).reshape(12, heads, 2, -1)[:n]
    assert np.array_equal(got[:, :, 0], fp4.encode(x[:, :heads].double().cpu().numpy()))
    assert np.array_equal(got[:, :, 1], fp4.encode(x[:, heads:].double().cpu().numpy()))
    before = cache.tensor.clone()
    cache.write(slots[:0], x[:0, :heads], x[:0, heads:])
    key, _ = cache.read(slots[:0], torch.bfloat16)
    assert key.shape == (0, heads, d) and torch.equal(cache.tensor, before)


# ---------------------------------------------------------------- attention
def filled(layout, bs, heads, d, lens, seed):
    """A cache whose rows hold no number but where a context's tokens are, its tables and the
    rows' oracle view."""
    g = torch.Generator().manual_seed(seed)
    pages = [-(-n // bs) for n in lens]
    blocks = sum(pages) + 3
    cache = Fp4Cache(torch.full(cache_shape(layout, blocks, bs, heads, d), 255, dtype=torch.uint8,
                                device="cuda"), d, layout)
    perm = torch.randperm(blocks, generator=g).int()
    width = max(1, max(pages)) + 1
    tables = torch.full((len(lens), width), 2 ** 30, dtype=torch.int32)
    slots, at = [], 0
    for s, n in enumerate(lens):
        tables[s, :pages[s]] = perm[at:at + pages[s]]
        at += pages[s]
        t = torch.arange(n)
        slots.append(tables[s][t // bs].long() * bs + t % bs)
    slots = torch.cat(slots)
    x = torch.randn(len(slots), heads, 2, d, generator=g)
    x[:, :, 0] *= 1 + 3 * (torch.rand(d, generator=g) > 0.9)
    if len(slots):
        cache.write(slots.cuda(), x[:, :, 0].cuda(), x[:, :, 1].cuda())
    return cache, tables


def check(cache, q, tables, lens, starts, scale, out, lse):
    """``out`` and ``lse`` against the oracle, within what the roundings may add up to.

    A score is a sum of d exact products in f32, in some order: off by at most
    (d + 4) 2^-24 sum |q_j k_j| scale, and by 2^-22 of itself from the scaling and the exponent's
    argument. A weight then is off by that, its exponential's 2^-22 and its rounding to bf16; the
    sums over n tokens and the joins add n 2^-24 of the weights' total."""
    d = q.shape[-1]
    want, wlse, reach, worst = fp4.attend(q.double().cpu().numpy(), canonical(cache), d,
                                          tables.cpu().numpy(), lens, starts, scale)
    n = max(lens) + 16
    score = (d + 4) * 2.0 ** -24 * worst + 2.0 ** -22 * worst + 2.0 ** -22
    weight = 2 * score + 2 * n * 2.0 ** -24
    room = reach * (weight[..., None] + 2.0 ** -8 * (1 + weight[..., None]))
    room += (np.abs(want) + room) * HALF_STEP[q.dtype] + 1e-30
    off = np.abs(out.double().cpu().numpy() - want)
    assert np.all(off <= room), float((off / room).max())
    if lse is not None:
        got = lse.double().cpu().numpy()
        empty = np.isneginf(wlse)
        assert np.array_equal(np.isneginf(got), empty)
        off = np.abs(got[~empty] - wlse[~empty])
        room = (weight + 2.0 ** -21 * (1 + np.abs(np.where(empty, 0, wlse))))[~empty]
        assert np.all(off <= room), float((off / room).max())


def attend_case(layout, bs, heads, shared, d, dtype, lens, news, seed=1, scale=None, **how):
    cache, tables = filled(layout, bs, heads, d, lens, seed)
    starts = np.concatenate(([0], np.cumsum(news)))
    g = torch.Generator().manual_seed(seed + 9)
    fused = torch.randn(int(starts[-1]), heads * shared + 2, d, generator=g).mul_(1.5)
    q = fused.to(TYPES[dtype]).cuda()[:, :heads * shared]
    given = dict(q_starts=torch.tensor(starts, dtype=torch.int32, device="cuda"), max_q=max(news))
    if all(n == 1 for n in news):
        given = dict()
    out, lse = cache.attend(q, tables.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"),
                            scale=scale, return_lse=True, **given, **how)
    check(cache, q, tables, lens, starts, scale or d ** -0.5, out, lse)


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("d", [16, 24, 32, 64, 72, 80, 96, 112, 120, 128, 136, 160, 192, 200, 256])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_single_tokens_over_every_head_size(ext, layout, d, dtype):
    attend_case(layout, 16, 2, 3, d, dtype, [1, 77, 300, 0, 33], [1] * 5, seed=d)


@pytest.mark.parametrize("bs", [1, 3, 8, 16, 24, 32, 48, 64, 128, 1000])
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 257, 1025])
def test_contexts_that_end_anywhere_in_a_tile_or_a_page(ext, bs, n):
    attend_case(LAYOUTS[n % 3], bs, 2, 2, 64, "bf16", [n, max(0, n - 1), n + 1], [1] * 3, seed=n)


@pytest.mark.parametrize("heads,shared", [(1, 1), (1, 8), (2, 7), (3, 16), (1, 17), (2, 40), (8, 4)])
@pytest.mark.parametrize("layout", LAYOUTS)
def test_heads_that_share(ext, heads, shared, layout):
    attend_case(layout, 16, heads, shared, 128, "bf16", [65, 200], [1, 1], seed=heads)


@pytest.mark.parametrize("d", [64, 80, 128, 192])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("bs", [16, 24])
def test_chunks_of_queries_see_what_is_before_them(ext, d, dtype, bs):
    # a whole prompt, a chunk after a prefix, single tokens, more queries than tokens (rows that see
    # nothing), an empty context with queries, a sequence without queries
    attend_case(LAYOUTS[d % 3], bs, 2, 4, d, dtype, [70, 150, 33, 5, 0, 40, 1, 260],
                [70, 37, 1, 9, 3, 0, 1, 130], seed=d)


@pytest.mark.parametrize("shared", [1, 5, 32])
@pytest.mark.parametrize("news", [[2, 3, 1], [17, 1, 64], [300, 129, 257]])
def test_few_and_many_queries_of_a_sequence(ext, shared, news):
    attend_case("combined", 32, 1, shared, 64, "bf16", [400, 131, 300], news, seed=shared)


@pytest.mark.parametrize("lens", [[4097], [9000, 3], [20000], [2500] * 3])
@pytest.mark.parametrize("news", [1, 4])
def test_long_contexts_are_split_and_joined(ext, lens, news):
    attend_case("combined", 16, 1, 4, 128, "bf16", lens, [news] * len(lens), seed=news)


def test_a_peaked_row_and_large_scores(ext):
    attend_case("kv_first", 16, 2, 4, 64, "bf16", [500, 90], [1, 1], scale=3.0)
    attend_case("kv_first", 16, 2, 4, 64, "f16", [500, 90], [40, 1], scale=0.001)


def test_pages_that_the_cache_does_not_have_hold_nothing(ext):
    for d, bs, news in ((64, 16, 1), (128, 24, 1), (128, 16, 40)):
        lens = [400, 130, 90]
        cache, tables = filled("kv_first", bs, 2, d, lens, 4)
        tables[0, 3], tables[0, 5], tables[0, 6] = -1, cache.num_blocks, -(2 ** 31)
        tables[1, 0] = 2 ** 31 - 1
        tables[2, :] = -5  # nothing at all
        starts = np.arange(0, 3 * news + 1, news)
        q = torch.randn(3 * news, 4, d, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
        out, lse = cache.attend(q, tables.cuda(), torch.tensor(lens).int().cuda(),
                                q_starts=torch.from_numpy(starts).int().cuda(), max_q=news,
                                return_lse=True)
        check(cache, q, tables, lens, starts, d ** -0.5, out, lse)
        assert torch.all(out[2 * news:] == 0) and torch.all(lse[2 * news:] == -math.inf)


def test_lengths_and_starts_past_their_arrays_are_cut(ext):
    cache, tables = filled("combined", 16, 1, 64, [64, 64], 5)
    tables = tables[:, :4].contiguous().cuda()  # room for 64 tokens
    q = torch.randn(4, 2, 64, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    lens = torch.tensor([10 ** 9, -7], dtype=torch.int32, device="cuda")
    out = cache.attend(q[:2], tables, lens)
    want = cache.attend(q[:2], tables, torch.tensor([64, 0], dtype=torch.int32, device="cuda"))
    assert torch.equal(out, want) and torch.all(out[1] == 0)
    starts = torch.tensor([-3, 2, 900], dtype=torch.int32, device="cuda")
    out = cache.attend(q, tables, torch.full((2,), 64).int().cuda(), q_starts=starts, max_q=4)
    good = torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    assert torch.equal(out, cache.attend(q, tables, torch.full((2,), 64).int().cuda(),
                                         q_starts=good, max_q=2))


def test_values_that_are_no_numbers_reach_only_the_rows_that_see_them(ext):
    cache, tables = filled("kv_first", 16, 1, 64, [100, 100], 6)
    x = torch.ones(1, 1, 64, device="cuda")
    x[0, 0, 40] = math.nan
    slot = tables[0, 5].long().reshape(1).cuda() * 16  # token 80 of the first sequence
    cache.write(slot, torch.ones_like(x), x)
    q = torch.randn(200, 2, 64, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    out = cache.attend(q, tables.cuda(), torch.tensor([100, 100]).int().cuda(),
                       q_starts=torch.tensor([0, 100, 200]).int().cuda(), max_q=100)
    bad = torch.isnan(out)
    assert not bad[:80].any() and not bad[100:].any()
    assert bad[80:100, :, 32:].all() and not bad[80:100, :, :32].any()


def test_pages_past_four_gigabytes(ext):
    # 2^32 bytes lie between the first page and the last
    heads, d, bs = 8, 256, 64
    blocks = (1 << 32) // (heads * bs * 2 * 136) + 9
    cache = Fp4Cache(torch.empty(cache_shape("combined", blocks, bs, heads, d), dtype=torch.uint8,
                                 device="cuda"), d, "combined")
    small = Fp4Cache.empty(3, bs, heads, d)
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(150, heads, 2, d, device="cuda", generator=g)
    q = torch.randn(1, 16, d, device="cuda", generator=g).bfloat16()
    outs = []
    for c, pages in ((cache, [blocks - 1, 0, blocks - 2]), (small, [0, 1, 2])):
        t = torch.arange(150, device="cuda")
        table = torch.tensor([pages], dtype=torch.int32, device="cuda")
        slots = table[0].long()[t // bs] * bs + t % bs
        c.write(slots, x[:, :, 0], x[:, :, 1])
        key, value = c.read(slots, torch.bfloat16)
        out = c.attend(q, table, torch.tensor([150], dtype=torch.int32, device="cuda"))
        outs.append((key, value, out))
    for a, b in zip(*outs):
        assert torch.equal(a, b)


def test_the_same_call_gives_the_same_bits_and_out_is_written_in_place(ext):
    cache, tables = filled("combined", 16, 2, 128, [5000, 900, 77], 8)
    q = torch.randn(3, 8, 128, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    lens = torch.tensor([5000, 900, 77], dtype=torch.int32, device="cuda")
    out = torch.full_like(q, 3.0)
    assert cache.attend(q, tables.cuda(), lens, out=out) is out
    for _ in range(3):
        assert torch.equal(cache.attend(q, tables.cuda(), lens), out)


def test_the_calls_run_on_the_current_stream(ext):
    cache, tables = filled("combined", 16, 2, 64, [3000, 200], 8)
    q = torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    lens = torch.tensor([3000, 200], dtype=torch.int32, device="cuda")
    dev = tables.cuda()
    want = cache.attend(q, dev, lens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [cache.attend(q, dev, lens) for _ in range(5)]
    others = [cache.attend(q, dev, lens) for _ in range(5)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs + others)


def test_a_captured_step_replays_with_new_rows(ext):
    """A decode step (the new rows written, then attention) in a graph, replayed with other rows
    between eager steps of the same shapes."""
    lens0 = [2000, 40, 700]
    caches = [filled("kv_first", 16, 2, 128, lens0, 8) for _ in range(2)]
    tables = caches[0][1].cuda()
    (graphed, _), (eager, _) = caches
    g = torch.Generator(device="cuda").manual_seed(5)
    key, value = (torch.randn(3, 2, 128, device="cuda", generator=g).bfloat16() for _ in range(2))
    q = torch.randn(3, 8, 128, device="cuda", generator=g).bfloat16()
    lens = torch.tensor(lens0, dtype=torch.int32, device="cuda")
    at = lens.long() - 1
    slots = tables.gather(1, (at // 16)[:, None])[:, 0].long() * 16 + at % 16

    def step(cache):
        cache.write(slots, key, value)
        return cache.attend(q, tables, lens)

    step(graphed)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(graphed)
    for _ in range(4):
        for t in (key, value, q):
            t.normal_(generator=g)
        graph.replay()
        want = step(eager)
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        assert torch.equal(graphed.tensor, eager.tensor)


def test_queries_that_want_a_gradient_are_refused(ext):
    cache, tables = filled("combined", 16, 1, 64, [10], 8)
    q = torch.zeros(1, 1, 64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    lens = torch.tensor([10], dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="backward"):
        cache.attend(q, tables.cuda(), lens)
    with torch.no_grad():
        assert torch.isfinite(cache.attend(q, tables.cuda(), lens)).all()
    with pytest.raises(RuntimeError, match="lengths"):
        cache.attend(q.detach(), tables.cuda(), lens.repeat(2))
    with pytest.raises(RuntimeError, match="query starts"):
        cache.attend(q.detach(), tables.cuda(), lens, q_starts=lens)
    with pytest.raises(RuntimeError, match="out must"):
        cache.attend(q.detach(), tables.cuda(), lens, out=torch.zeros(1, 1, 64, device="cuda"))
    with pytest.raises(RuntimeError, match="int32"):
        cache.attend(q.detach(), tables.cuda().long(), lens)


# ---------------------------------------------------------------- how the work is dealt out
@pytest.mark.parametrize("heads", [1, 2, 3, 5, 6, 7, 8, 10, 12])
@pytest.mark.parametrize("layout", LAYOUTS)
def test_heads_that_lie_side_by_side_are_taken_together(ext, heads, layout):
    # enough sequences that a workgroup takes as many heads as it can; lengths about a stage's and a
    # share's ends
    lens = [0, 1, 31, 32, 33, 255, 256, 257, 511, 513, 640, 7] * 10
    attend_case(layout, 16, heads, 1, 32, "bf16", lens, [1] * len(lens), seed=heads, max_len=4096)


@pytest.mark.parametrize("d,dtype", [(24, "f16"), (96, "bf16"), (128, "f16"), (192, "bf16"),
                                     (256, "f16")])
def test_tiles_in_several_shares_of_unlike_sequences(ext, d, dtype):
    # shares that end in a tile, in the next one and at a tile's start
    lens = [5000, 3, 0, 1300, 1024, 2048, 1, 700, 3333]
    attend_case("kv_first", 16, 2, 2, d, dtype, lens, [1] * len(lens), seed=d)
    attend_case("combined", 24, 1, 3, d, dtype, lens, [7, 3, 2, 11, 1, 5, 1, 16, 4], seed=d)


@pytest.mark.parametrize("d,dtype", [(64, "bf16"), (72, "f16"), (128, "bf16"), (200, "f16")])
def test_long_chunks_are_split_too(ext, d, dtype):
    attend_case("kv_first", 16, 1, 5, d, dtype, [2100, 1500, 90, 4000], [40, 130, 90, 14], seed=d)


@pytest.mark.parametrize("d,dtype", [(64, "f16"), (128, "bf16"), (192, "bf16")])
@pytest.mark.parametrize("seqs,max_len", [(5, 0), (300, 0), (300, 1 << 20)])
def test_65_to_128_query_rows_of_a_head(ext, d, dtype, seqs, max_len):
    # the rows go to either kernel by how much there is to do, up to the tables' room
    lens = [1100] + [40 + 7 * (i % 9) for i in range(seqs - 1)]
    news = [[26, 32, 17, 33, 1][i % 5] for i in range(seqs)]
    attend_case("blocks_first", 16, 1, 4, d, dtype, lens, news, seed=d, max_len=max_len)


@pytest.mark.parametrize("seqs", [257, 513, 1100])
def test_more_sequences_than_a_workgroup_has_threads(ext, seqs):
    lens = [(37 * i) % 90 for i in range(seqs)]
    lens[seqs // 2], lens[-1] = 1500, 1100
    attend_case("combined", 16, 1, 2, 16, "bf16", lens, [1] * seqs, seed=seqs)
    news = [1 + (i % 3) * 20 for i in range(seqs)]
    attend_case("kv_first", 16, 1, 2, 16, "bf16", lens, news, seed=seqs)
    attend_case("kv_first", 16, 1, 2, 16, "bf16", [min(n, 80) for n in lens], news, seed=seqs)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("news,shared", [(3, 4), (16, 1), (100, 2), (33, 5)])
@pytest.mark.parametrize("back", [0, 1, 2])
def test_no_number_in_a_masked_place(ext, d, news, shared, back):
    """A token whose V holds a group without a number, at the last places of a chunk: the rows before
    it are as without it, in the same products' tile."""
    n = 200
    cache, tables = filled("kv_first", 16, 1, d, [n, n], 6)
    at = n - 1 - back
    x = torch.ones(1, 1, d, device="cuda")
    x[0, 0, d - 10] = math.inf
    slot = tables[0, at // 16].long().reshape(1).cuda() * 16 + at % 16
    q = torch.randn(2 * news, shared, d, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    how = dict(q_starts=torch.tensor([0, news, 2 * news]).int().cuda(), max_q=news)
    lens = torch.tensor([n, n], device="cuda").int()
    ones = torch.ones_like(x)
    cache.write(slot, ones, ones)
    want = cache.attend(q, tables.cuda(), lens, **how)
    cache.write(slot, ones, x)
    out = cache.attend(q, tables.cuda(), lens, **how)
    hit = news - 1 - back  # the first query that sees the token
    bad = torch.isnan(out)
    rows = slice(max(hit, 0), news)
    group = slice((d - 10) // 32 * 32, min(d, (d - 10) // 32 * 32 + 32))
    assert bad[rows, :, group].all()
    bad[rows, :, group] = False
    assert not bad.any()
    same = torch.ones_like(bad)
    same[rows, :, group] = False
    assert torch.equal(out[same], want[same])
    # and a K without a number: the rows that see it are none, the others as they were
    cache.write(slot, x, ones)
    out = cache.attend(q, tables.cuda(), lens, **how)
    assert torch.isnan(out[rows]).all() and torch.equal(out[:rows.start], want[:rows.start])
    assert torch.equal(out[news:], want[news:])


def test_padding_queries_that_no_sequence_names_are_left_alone(ext):
    cache, tables = filled("kv_first", 16, 1, 64, [300, 40], 6)
    q = torch.randn(90, 4, 64, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    lens = torch.tensor([300, 40]).int().cuda()
    for starts in ([0, 1, 31], [3, 60, 62], [10, 10, 50]):
        out = torch.full_like(q, 7.0)
        cache.attend(q, tables.cuda(), lens, q_starts=torch.tensor(starts).int().cuda(), max_q=60,
                     out=out)
        assert torch.all(out[:starts[0]] == 7) and torch.all(out[starts[2]:] == 7)
        part = q[starts[0]:starts[2]].contiguous()
        own = torch.tensor([s - starts[0] for s in starts]).int().cuda()
        want = cache.attend(part, tables.cuda(), lens, q_starts=own, max_q=60)
        assert torch.equal(out[starts[0]:starts[2]], want)


def test_a_captured_batch_replays_with_other_lengths(ext):
    """The shares are found on the device: a graph holds for any lengths."""
    lens0 = [3000, 40, 700, 0]
    cache, tables = filled("combined", 16, 2, 64, [4000, 900, 900, 900], 8)
    dev = tables.cuda()
    g = torch.Generator(device="cuda").manual_seed(5)
    q = torch.randn(90, 8, 64, device="cuda", generator=g).bfloat16()
    lens = torch.tensor(lens0, dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 1, 2, 80, 81], dtype=torch.int32, device="cuda")

    def step():
        return cache.attend(q, dev, lens, q_starts=starts, max_q=80, return_lse=True)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for new, at in (([3000, 40, 700, 0], [0, 1, 2, 80, 81]), ([4000, 900, 80, 3], [0, 9, 10, 11, 90]),
                    ([1, 2, 3, 4], [0, 1, 2, 3, 4]), ([0, 0, 900, 900], [0, 80, 81, 82, 90])):
        lens.copy_(torch.tensor(new, dtype=torch.int32))
        starts.copy_(torch.tensor(at, dtype=torch.int32))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        n = at[-1]
        assert torch.equal(got[0][:n], want[0][:n]) and torch.equal(got[1][:n], want[1][:n])
