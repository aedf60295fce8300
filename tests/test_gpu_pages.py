"""Pages copied and packed on the GPU against the oracle, and the 4-bit path end to end: written,
attended, forked, packed, taken as a snapshot and put back."""

import numpy as np
import pytest
import torch

from everserve_amd.state.fp4 import Fp4Cache, row_bytes
from everserve_amd.state.pages import PageMover
from everserve_amd.state.paged import PagedKV
from oracle import fp4
from tests.cases import LAYOUTS, bits, caches

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def pages_of(layer, layout):
    return layer.transpose(0, 1) if layout == "kv_first" else layer


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("d", [1, 6, 8, 36, 64])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.uint8, torch.float32])
def test_pages_are_copied_whole_in_every_layer(ext, layout, d, dtype):
    cpu = caches(layout, d, torch.bfloat16, n_layers=3, seed=d)
    cpu = [(t.float() * 50).to(dtype) for t in cpu]
    gpu = [t.cuda() for t in cpu]
    blocks = pages_of(cpu[0], layout).shape[0]
    src, dst = [0, 3, -1, 2, blocks, 5, 1], [4, 6, 1, blocks, 2, 5, -7]  # two pairs move a page
    PageMover(gpu, layout).copy(ints(src), ints(dst))
    for t in cpu:
        p = pages_of(t, layout)
        p[4], p[6] = p[0].clone(), p[3].clone()
    torch.cuda.synchronize()
    for a, b in zip(gpu, cpu):
        assert np.array_equal(bits(a), bits(b))


@pytest.mark.parametrize("layout", LAYOUTS)
def test_a_view_of_some_heads_moves_alone_and_a_count_cuts_the_list(ext, layout):
    gpu = [t.cuda() for t in caches(layout, 8, torch.bfloat16, n_layers=2, seed=4)]
    want = [t.clone() for t in gpu]
    heads = slice(1, 3)
    view = [t[:, heads] if layout == "combined" else t[..., heads, :] for t in gpu]
    for count, moves in ((0, 0), (1, 1), (9, 2), (-3, 0)):
        PageMover(view, layout).copy(ints([5, 6]), ints([1, 2]), ints([count]))
        for t in want:
            p = pages_of(t, layout)
            for s, d in ((5, 1), (6, 2))[:moves]:
                if layout == "combined":
                    p[d, heads] = p[s, heads].clone()
                else:
                    p[d, ..., heads, :] = p[s, ..., heads, :].clone()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(gpu, want))


@pytest.mark.parametrize("blocks,rows,width", [(1, 1, 1), (2, 3, 2), (31, 4, 9), (32, 4, 9),
                                               (33, 7, 5), (100, 16, 1), (1000, 30, 40),
                                               (4096, 64, 33), (70001, 300, 97), (300000, 9, 20000)])
@pytest.mark.parametrize("share", [0.0, 0.5, 1.0])
def test_a_plan_is_the_oracles(ext, blocks, rows, width, share):
    g = np.random.default_rng(blocks + rows)
    top = max(1, int(blocks * (0.3 + 0.7 * share)))
    tables = g.integers(-2, top + (2 if share == 1 else 0), (rows, width)).astype(np.int32)
    counts = g.integers(-1, width + 2, rows).astype(np.int32)
    if share == 0:
        counts[:] = 0  # nothing in use
    dev = torch.from_numpy(np.pad(tables, ((0, 0), (0, 3)))).cuda()[:, :width]  # rows apart
    got = ext.plan_compaction(dev, torch.from_numpy(counts).cuda(), blocks)
    want, moves, used = fp4.plan_compaction(tables, np.minimum(counts, width), blocks)
    assert got[3].tolist() == [used, len(moves)]
    assert np.array_equal(got[0].cpu().numpy(), np.array(want, dtype=np.int32).reshape(rows, width))
    pad = [-1] * (blocks // 2 - len(moves))
    assert got[1].tolist() == [a for a, _ in moves] + pad
    assert got[2].tolist() == [b for _, b in moves] + pad
    if share == 1:  # without counts every entry is in use
        got = ext.plan_compaction(dev, None, blocks)
        _, moves, used = fp4.plan_compaction(tables, [width] * rows, blocks)
        assert got[3].tolist() == [used, len(moves)]


def test_no_tables_and_no_pages(ext):
    empty = torch.zeros((0, 5), dtype=torch.int32, device="cuda")
    got = ext.plan_compaction(empty, None, 10)
    assert got[3].tolist() == [0, 0] and got[1].tolist() == [-1] * 5 and got[0].shape == (0, 5)
    got = ext.plan_compaction(ints([[3, 1]]), None, 0)
    assert got[3].tolist() == [0, 0] and got[0].tolist() == [[3, 1]]


@pytest.mark.parametrize("layout", LAYOUTS)
def test_a_packed_cache_holds_the_same_rows_under_its_new_tables(ext, layout):
    g = torch.Generator(device="cuda").manual_seed(3)
    blocks, bs, heads, d = 200, 4, 2, 24
    shape = {"kv_first": (2, blocks, bs, heads, d), "blocks_first": (blocks, 2, bs, heads, d),
             "combined": (blocks, heads, bs, 2 * d)}[layout]
    layers = [torch.randn(shape, device="cuda", generator=g).bfloat16() for _ in range(5)]
    before = [pages_of(t, layout).clone() for t in layers]
    perm = torch.randperm(blocks, device="cuda", generator=g).int()
    tables = perm[:90].reshape(6, 15).contiguous()
    tables[3, :5] = tables[0, :5]  # a shared prefix
    kept = tables.clone()
    plan = PageMover(layers, layout).compact(tables)
    used, moved = plan.sizes.tolist()
    assert torch.equal(tables, kept) and used == 85 and moved > 0
    assert int(plan.tables.max()) == used - 1
    for a, b in zip(layers, before):
        assert torch.equal(pages_of(a, layout)[plan.tables.long()], b[kept.long()])


def test_a_plan_and_its_copy_replay_in_a_graph(ext):
    g = torch.Generator(device="cuda").manual_seed(3)
    layers = [torch.randint(0, 255, (300, 2, 16, 72), dtype=torch.uint8, device="cuda")
              for _ in range(3)]
    mover = PageMover(layers, "combined")
    tables = torch.randperm(300, device="cuda", generator=g).int()[:120].reshape(8, 15).contiguous()
    mover.compact(tables)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan = mover.compact(tables)
    for _ in range(4):
        tables.copy_(torch.randperm(300, device="cuda", generator=g).int()[:120].reshape(8, 15))
        before = [t.clone() for t in layers]
        graph.replay()
        want = mover.plan(tables)
        torch.cuda.synchronize()
        for f in ("tables", "src", "dst", "sizes"):
            assert torch.equal(getattr(plan, f), getattr(want, f))
        for a, b in zip(layers, before):
            assert torch.equal(a[plan.tables.long()], b[tables.long()])


def test_a_four_bit_rank_is_forked_packed_and_restored(ext):
    """The path as a rank runs it: prompts written and attended over, a sequence forked, the cache
    packed, its rows gathered as the snapshot gathers them and scattered into a spare's caches at
    other slots, with the same attention at each stage."""
    g = torch.Generator(device="cuda").manual_seed(9)
    n_layers, blocks, bs, heads, shared, d = 3, 60, 16, 2, 4, 128
    rank = [Fp4Cache.empty(blocks, bs, heads, d, "kv_first") for _ in range(n_layers)]
    perm = torch.randperm(blocks, device="cuda", generator=g).int()
    lens = ints([150, 90, 31])
    tables = torch.full((4, 11), -1, dtype=torch.int32, device="cuda")
    counts = [10, 6, 2]
    for s, c in enumerate(counts):
        tables[s, :c] = perm[sum(counts[:s]):sum(counts[:s + 1])]
    q = torch.randn(4, heads * shared, d, device="cuda", generator=g).bfloat16()
    for c in rank:
        for s in range(3):
            t = torch.arange(int(lens[s]), device="cuda")
            slots = tables[s][t // bs].long() * bs + t % bs
            x = torch.randn(2, len(t), heads, d, device="cuda", generator=g).bfloat16()
            c.write(slots, x[0], x[1])

    # the fourth sequence parts from the first: it shares all pages but the last, which it copies
    tables[3] = tables[0]
    tables[3, 9] = perm[30]
    mover = PageMover([c.tensor for c in rank], "kv_first")
    mover.copy(tables[0, 9:10].contiguous(), tables[3, 9:10].contiguous())
    lens = ints([150, 90, 31, 150])
    want = [c.attend(q, tables, lens) for c in rank]
    for c, w in zip(rank, want):
        again = c.attend(q[[0, 1, 2, 0]].contiguous(), tables, lens)
        assert torch.equal(again[3], w[0])

    plan = mover.compact(tables, ints([10, 6, 2, 10]))
    used = int(plan.sizes[0])
    assert used == 19
    for c, w in zip(rank, want):
        assert torch.equal(c.attend(q, plan.tables, lens), w)

    # every used slot of every layer to staging rows and back, at other slots of fresh caches
    paged = PagedKV.of(rank[0].tensor)
    half = row_bytes(d)
    n = used * bs
    rows = torch.empty(n_layers, heads, n, 2, half, dtype=torch.uint8, device="cuda")
    ids = torch.arange(n, device="cuda")
    held = torch.arange(heads, device="cuda")

    def table_of(cs):
        return torch.tensor([c.tensor.data_ptr() for c in cs], device="cuda")

    ext.gather_rows(table_of(rank), ids, held, rows.data_ptr(), n, half, bs,
                    paged.layout_strides(rank[0].tensor), 1)
    spare = [Fp4Cache.empty(blocks, bs, heads, d, "kv_first") for _ in range(n_layers)]
    to = torch.randperm(blocks, device="cuda", generator=g)[:used]
    slots = (to[:, None] * bs + torch.arange(bs, device="cuda")).reshape(-1)
    ext.scatter_rows(table_of(spare), slots, held, rows.data_ptr(), n, half, bs,
                     paged.layout_strides(spare[0].tensor), 1)
    moved = torch.where(plan.tables >= 0, to[plan.tables.clamp(0, used - 1).long()].int(),
                        plan.tables)
    for c, w in zip(spare, want):
        assert torch.equal(c.attend(q, moved, lens), w)
