"""Attention behind a shared prefix, eviction by the weights that it gave, and compaction, as a server
runs them: prompts in chunks, steps of single tokens, sequences cut short, and steps after that."""

import numpy as np
import pytest
import torch

from everserve_amd.state.evict import Evictor
from everserve_amd.state.full import FullCache, SharedPrefix
from oracle import full
from tests.test_gpu_full import compare, compare_mass

pytestmark = pytest.mark.gpu

LAYERS, BLOCKS, BS, HEADS, SHARED, D = 2, 64, 16, 2, 4, 64
PREFIX, BUDGET, RECENT = 40, 48, 16


def ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


class Server:
    """Three sequences, of which the first two share a prefix, with pages dealt from the far end."""

    def __init__(self, layout, dtype):
        shape = {"kv_first": (2, BLOCKS, BS, HEADS, D), "combined": (BLOCKS, HEADS, BS, 2 * D)}
        self.g = torch.Generator().manual_seed(3)
        self.dtype, self.layout = dtype, layout
        self.caches = [FullCache(torch.full(shape[layout], float("nan"), dtype=dtype).cuda(), layout)
                       for _ in range(LAYERS)]
        self.mass = torch.zeros(LAYERS, BLOCKS, HEADS, BS, device="cuda")
        self.evictor = Evictor([c.tensor for c in self.caches], layout)
        self.free = list(range(BLOCKS))
        self.prefix_table = [[self.free.pop() for _ in range(3)]]
        self.tables = [[self.free.pop() for _ in range(7)] for _ in range(3)]
        self.lens = [0, 0, 0]
        self.write(self.prefix_table[0], 0, PREFIX)

    def write(self, table, first, n):
        for c in self.caches:
            x = torch.randn(n, HEADS, 2, D, generator=self.g).to(self.dtype).cuda()
            t = np.arange(first, first + n)
            page, off = np.array(table)[t // BS].tolist(), (t % BS).tolist()
            if self.layout == "combined":
                c.tensor[page, :, off] = x.reshape(n, HEADS, 2 * D)
            else:
                c.tensor[:, page, off] = x.permute(2, 0, 1, 3)

    def step(self, news):
        """New tokens of each sequence, and every layer's attention over them and what it holds."""
        for s, n in enumerate(news):
            self.write(self.tables[s], self.lens[s], n)
            self.lens[s] += n
        starts = np.concatenate(([0], np.cumsum(news)))
        how = {} if max(news) == 1 else dict(q_starts=ints(starts), max_q=max(news))
        prefix = SharedPrefix(ints(self.prefix_table), ints([PREFIX]), ints([0, 2]))
        plain = (np.array(self.prefix_table), [PREFIX], [0, 2])
        for la, c in enumerate(self.caches):
            q = torch.randn(sum(news), HEADS * SHARED, D, generator=self.g).to(self.dtype).cuda()
            before = self.mass[la].double().cpu().numpy()
            out, lse = c.attend(q, ints(self.tables), ints(self.lens), return_lse=True,
                                prefix=prefix, mass=self.mass[la], **how)
            view = full.canonical(c.tensor.double().cpu().numpy(), self.layout)
            want = full.attend(q.double().cpu().numpy(), view, np.array(self.tables), self.lens,
                               starts, D ** -0.5, plain, before)
            longest = PREFIX + max(self.lens)
            compare(want, D, self.dtype, longest, out, lse)
            compare_mass(want, before, D, sum(news) * SHARED, longest, self.mass[la])

    def evict(self):
        room = BUDGET // BS
        new = [[self.free.pop(0) for _ in range(room)] for _ in range(3)]
        views = [full.canonical(c.tensor.float().cpu().numpy(), self.layout) for c in self.caches]
        mass = self.mass.cpu().numpy().copy()
        lens, kept = full.evict(views, mass, np.array(self.tables), self.lens, np.array(new),
                                BUDGET, RECENT)
        got = self.evictor.evict(ints(self.tables), ints(self.lens), ints(new), BUDGET, self.mass,
                                 recent=RECENT)
        assert np.array_equal(got.lens.cpu().numpy(), lens)
        assert np.array_equal(got.kept.cpu().numpy(), kept)
        assert np.array_equal(self.mass.cpu().numpy(), mass)
        for c, w in zip(self.caches, views):
            assert np.array_equal(full.canonical(c.tensor.float().cpu().numpy(), self.layout), w,
                                  equal_nan=True)
        for s in range(3):
            self.free += self.tables[s]
            self.tables[s] = new[s] + [self.free.pop(0) for _ in range(2)]
        self.lens = lens.tolist()

    def compact(self):
        every = ints([self.prefix_table[0] + [0, 0]] + self.tables)
        done = self.evictor.compact(every, ints([3] + [5] * 3))
        used, moved = done.sizes.tolist()
        assert used == 3 + 3 * 5 and moved > 0
        src, dst = done.src[:moved].long(), done.dst[:moved].long()
        self.mass[:, dst] = self.mass[:, src]
        rows = done.tables.tolist()
        self.prefix_table, self.tables = [rows[0][:3]], rows[1:]
        assert max(max(r) for r in self.prefix_table + self.tables) < used
        self.free = list(range(used, BLOCKS))


@pytest.mark.parametrize("layout,dtype", [("kv_first", torch.bfloat16),
                                          ("combined", torch.float16)])
def test_prompts_steps_eviction_and_compaction_in_a_row(ext, layout, dtype):
    server = Server(layout, dtype)
    server.step([70, 50, 33])  # prompts, in two chunks
    server.step([20, 1, 30])
    server.step([1, 1, 1])
    server.evict()
    server.step([1, 1, 1])
    server.step([1, 1, 1])
    server.compact()
    server.step([1, 1, 1])
    server.step([9, 1, 12])
    server.evict()  # of 60, 52 and 63
    server.step([1, 1, 1])


def test_an_eviction_behind_attention_on_another_stream(ext):
    """Attention, eviction and attention again, enqueued on a stream without a wait in between."""
    server = Server("kv_first", torch.bfloat16)
    server.step([90, 80, 60])
    c, mass = server.caches[0], server.mass[:1]
    q = torch.randn(3, HEADS * SHARED, D, generator=server.g).bfloat16().cuda()
    new = ints([[server.free.pop(0) for _ in range(3)] for _ in range(3)])
    tables, lens = ints(server.tables), ints(server.lens)
    evictor = Evictor([c.tensor], "kv_first")

    def run(mass):
        first = c.attend(q, tables, lens, mass=mass[0])
        done = evictor.evict(tables, lens, new, BUDGET, mass, recent=RECENT)
        return first, c.attend(q, new, done.lens, mass=mass[0]), done.kept

    want_mass, got_mass = mass.clone(), mass.clone()
    want = run(want_mass)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = run(got_mass)
    stream.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert torch.equal(got_mass, want_mass)


@pytest.mark.parametrize("max_len", [1, 16, 40, 100])
def test_weights_where_the_bound_is_below_the_lengths(ext, max_len):
    """Tokens past the bound have no score kept for them; their weights are the same."""
    server = Server("kv_first", torch.bfloat16)
    server.step([90, 80, 60])
    c = server.caches[0]
    q = torch.randn(3, HEADS * SHARED, D, generator=server.g).bfloat16().cuda()
    before = server.mass[0].double().cpu().numpy()
    mass = server.mass[0].clone()
    out, lse = c.attend(q, ints(server.tables), ints(server.lens), return_lse=True, mass=mass,
                        max_len=max_len)
    view = full.canonical(c.tensor.double().cpu().numpy(), "kv_first")
    want = full.attend(q.double().cpu().numpy(), view, np.array(server.tables), server.lens,
                       np.arange(4), D ** -0.5, None, before)
    compare(want, D, torch.bfloat16, 90, out, lse)
    compare_mass(want, before, D, SHARED, 90, mass)
