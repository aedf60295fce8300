"""The weights of tokens on the GPU where a wave, a workgroup or a call takes them in turns: rounds of
tokens, and more query heads on a KV head than share a prefix's tiles."""

import math

import pytest
import torch

from tests.test_gpu_full import Batch, ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,dtype", [(64, "bf16"), (80, "f16"), (128, "bf16"), (192, "f16")])
@pytest.mark.parametrize("news,shared", [(4, 5), (9, 7), (16, 4), (40, 3)])
@pytest.mark.parametrize("before", [0, 1100])
def test_a_waves_tokens_in_several_rounds(ext, d, dtype, news, shared, before):
    """A bound far below the lengths leaves one workgroup all of a context's rounds: 20 and 63 rows,
    of which each wave has tokens of its own, and 64 and more, which the waves share."""
    Batch("kv_first", 16, 1, shared, d, dtype, [1500], [news], seed=news,
          prefixes=[before] if before else [], groups=[0, 1]).check(max_len=1, prefix_len=1)


@pytest.mark.parametrize("d,dtype", [(64, "bf16"), (128, "f16"), (192, "bf16")])
@pytest.mark.parametrize("heads,shared", [(1, 65), (1, 71), (2, 96), (1, 128)])
def test_more_heads_than_share_a_prefixs_tiles(ext, d, dtype, heads, shared):
    """Beyond 64 query heads a KV head even one token takes its group's prefix by itself."""
    Batch("kv_first", 16, heads, shared, d, dtype, [65, 20, 1, 0], [1] * 4, seed=shared,
          prefixes=[99, 30], groups=[0, 2, 4]).check()
    Batch("combined", 16, heads, shared, d, dtype, [65, 20, 3], [5, 1, 4], seed=shared,
          prefixes=[99], groups=[0, 2]).check()


@pytest.mark.parametrize("held", [math.nan, -60.0, 0.0])
@pytest.mark.parametrize("shared", [1, 4, 64, 65, 71])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_queries_that_are_not_taken_weigh_nothing_whatever_the_memory_held(ext, held, shared, dtype):
    """Queries past max_q and between sequences: a prefix's tokens get nothing of them."""
    b = Batch("kv_first", 16, 1, shared, 64, dtype, [300, 40], [45, 45], seed=6, prefixes=[100],
              groups=[0, 2])
    lens, tables, prefix = ints([300, 40]), b.tables.cuda(), b.prefix()
    starts, max_q = ints([3, 45, 88]), 20
    kept = torch.cat((torch.arange(3, 23), torch.arange(45, 65))).cuda()
    mass, own_mass = b.mass.clone(), b.mass.clone()
    want = b.cache.attend(b.q[kept].contiguous(), tables, lens, q_starts=ints([0, 20, 40]),
                          max_q=20, prefix=prefix, mass=own_mass)
    for _ in range(3):
        blocks = [torch.full((1 << 20,), held, device="cuda") for _ in range(24)]
        blocks += [torch.full((1 << n,), held, device="cuda") for n in range(7, 19) for _ in range(4)]
        torch.cuda.synchronize()
        del blocks
        mass.copy_(b.mass)
        out = b.cache.attend(b.q, tables, lens, q_starts=starts, max_q=max_q, prefix=prefix,
                             mass=mass)
        assert torch.equal(out[kept], want)
        # The rows lie in other tiles of 16: the same weights in another order of sums. Up to 2,840
        # rows go to 4 waves of 16 lanes, so a sum has 45 terms, 4 and 3 joins and the old mass: off
        # by 53 times 2^-24 on either side, 6.4e-6 of it.
        assert torch.allclose(mass, own_mass, rtol=1e-5, atol=0)
