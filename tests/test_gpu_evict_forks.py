"""Masses beside pages that are copied or filled: what a caller moves with them, and what an eviction
then goes by."""

import pytest
import torch

from everserve_amd.state.evict import Evictor
from tests.test_gpu_full import ints

pytestmark = pytest.mark.gpu

LAYERS, BLOCKS, HEADS, BS, D = 2, 24, 3, 16, 32


def cache(g):
    return [torch.randn(2, BLOCKS, BS, HEADS, D, device="cuda", generator=g).bfloat16()
            for _ in range(LAYERS)]


def test_a_forks_masses_go_with_its_pages(ext):
    """A sequence forks inside its last page: with that page's masses both forks keep the same
    tokens and rows, and without them the copy's are another's."""
    g = torch.Generator(device="cuda").manual_seed(1)
    layers = cache(g)
    evictor = Evictor(layers, "kv_first")
    mass = torch.rand(LAYERS, BLOCKS, HEADS, BS, device="cuda", generator=g)
    mass[:, 7] += 10  # another sequence's, from before
    tables = ints([[0, 1, 2], [0, 1, 7]])
    evictor.copy(ints([2]), ints([7]))
    stale = evictor.evict(tables, ints([45, 45]), ints([[8, 9], [10, 11]]), 20, mass.clone(), recent=4)
    assert not torch.equal(stale.kept[:, 0], stale.kept[:, 1])
    mass[:, 7] = mass[:, 2]
    done = evictor.evict(tables, ints([45, 45]), ints([[8, 9], [10, 11]]), 20, mass, recent=4)
    assert torch.equal(done.kept[:, 0], done.kept[:, 1]) and done.lens.tolist() == [20, 20]
    for t in layers:
        assert torch.equal(t[:, 8], t[:, 10]) and torch.equal(t[:, 9, :4], t[:, 11, :4])
    assert torch.equal(mass[:, 8], mass[:, 10]) and torch.equal(mass[:, 9, :, :4], mass[:, 11, :, :4])


def test_restored_pages_begin_at_no_mass(ext):
    """Pages filled from elsewhere hold the masses of whatever was there: cleared, the newest and the
    first of the others stay."""
    g = torch.Generator(device="cuda").manual_seed(2)
    evictor = Evictor(cache(g), "kv_first")
    mass = torch.rand(LAYERS, BLOCKS, HEADS, BS, device="cuda", generator=g)
    pages = [3, 4, 5]
    mass[:, pages] = 0
    done = evictor.evict(ints([pages]), ints([40]), ints([[6]]), 16, mass, recent=6)
    want = torch.cat((torch.arange(10), torch.arange(34, 40))).int().cuda()
    assert torch.equal(done.kept, want.expand(LAYERS, 1, HEADS, 16))


def test_tokens_on_pages_outside_count_and_leave_their_new_slots(ext):
    """Fewer tokens than the budget on pages that there are: the others stay in the length, and
    their new slots hold what they held."""
    g = torch.Generator(device="cuda").manual_seed(3)
    layers = cache(g)
    before = [t.clone() for t in layers]
    mass = torch.rand(LAYERS, BLOCKS, HEADS, BS, device="cuda", generator=g)
    held = mass.clone()
    done = Evictor(layers, "kv_first").evict(ints([[0, -1]]), ints([30]), ints([[8, 9]]), 30, mass)
    assert done.lens.tolist() == [30]
    for t, b in zip(layers, before):
        assert torch.equal(t[:, 8], b[:, 0]) and torch.equal(t[:, 9], b[:, 9])
    assert torch.equal(mass[:, 8], held[:, 0]) and torch.equal(mass[:, 9], held[:, 9])
