"""The 4-bit cache's calls and the page moves on a stream of their own: each must be ordered behind
what was queued there before it, the work that makes its inputs."""

import pytest
import torch

from everserve_amd.state.fp4 import Fp4Cache
from everserve_amd.state.pages import PageMover
from tests.test_gpu_fp4 import filled

pytestmark = pytest.mark.gpu


def ints(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.fixture
def behind(ext):
    """``behind(inputs, news, call)``: ``call`` on a side stream, behind milliseconds of products and
    the copies of ``news`` into ``inputs``, which hold other values until then. A call on any other
    stream reads those."""
    a = torch.randn(8192, 8192, device="cuda", dtype=torch.bfloat16)
    b = torch.empty_like(a)  # kept: nothing of the call's is to share memory with the products
    torch.cuda.synchronize()

    def run(inputs, news, call):
        side = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            for _ in range(8):
                torch.mm(a, a, out=b)
            for x, new in zip(inputs, news):
                x.copy_(new)
            got = call()
        side.synchronize()
        return got

    return run


@pytest.mark.parametrize("news", [1, 40])
def test_attention_waits_for_its_stream(behind, news):
    cache, tables = filled("kv_first", 16, 2, 128, [3000, 200, 77], 8)
    tables = tables.cuda()
    starts = torch.arange(0, 3 * news + 1, news, dtype=torch.int32, device="cuda")
    how = dict(q_starts=starts, max_q=news, return_lse=True)
    q, new_q = (torch.randn(3 * news, 8, 128, device="cuda").bfloat16() for _ in range(2))
    lens, new_lens = ints(3000, 200, 77), ints(2999, 150, 60)
    got = behind((q, lens), (new_q, new_lens), lambda: cache.attend(q, tables, lens, **how))
    want = cache.attend(new_q, tables, new_lens, **how)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_rows_are_written_and_read_in_their_stream(behind):
    caches = [Fp4Cache.empty(8, 16, 2, 64) for _ in range(2)]
    rows, new = (torch.randn(2, 100, 2, 64, device="cuda").bfloat16() for _ in range(2))
    slots = torch.randperm(128, device="cuda")[:100]
    behind((rows,), (new,), lambda: caches[0].write(slots, rows[0], rows[1]))
    caches[1].write(slots, new[0], new[1])
    torch.cuda.synchronize()
    assert torch.equal(caches[0].tensor, caches[1].tensor)
    old = caches[0].tensor.clone()
    changed = old.flip(0).contiguous()
    got = behind((caches[0].tensor,), (changed,), lambda: caches[0].read(slots, torch.bfloat16))
    caches[1].tensor.copy_(changed)
    want = caches[1].read(slots, torch.bfloat16)
    assert all(torch.equal(torch.nan_to_num(a), torch.nan_to_num(b)) for a, b in zip(got, want))


def test_pages_are_copied_and_packed_in_their_stream(behind):
    layers = [torch.randint(0, 255, (300, 2, 16, 72), dtype=torch.uint8, device="cuda")
              for _ in range(3)]
    mover = PageMover(layers, "combined")
    src, dst, new_src = ints(1, 2, 3), ints(200, 201, 202), ints(7, 8, 9)
    before = [t.clone() for t in layers]
    behind((src,), (new_src,), lambda: mover.copy(src, dst))
    for t, old in zip(layers, before):
        assert torch.equal(t[200:203], old[7:10])

    tables = torch.randperm(300, device="cuda").int()[:120].reshape(8, 15).contiguous()
    new = torch.randperm(300, device="cuda").int()[:120].reshape(8, 15).contiguous()
    before = [t.clone() for t in layers]
    plan = behind((tables,), (new,), lambda: mover.compact(tables))
    want = mover.plan(new)
    assert torch.equal(plan.tables, want.tables) and torch.equal(plan.sizes, want.sizes)
    for t, old in zip(layers, before):
        assert torch.equal(t[plan.tables.long()], old[new.long()])
