"""Attention over the longest context that there may be, 2^31 - 1 tokens, whose pages are one page over
and over: tokens are numbered in 32 bits up to its end."""

import math

import pytest
import torch

from everserve_amd.state.full import FullCache
from tests.test_gpu_full import ints

pytestmark = pytest.mark.gpu

BS, PAGES = 1 << 20, 1 << 11


@pytest.mark.parametrize("news", [1, 5, 40])
def test_the_last_of_the_longest_contexts_tokens(ext, news):
    """The last token's V holds no number, and the row of it alone sees that."""
    cache = torch.zeros(2, 2, BS, 1, 16, dtype=torch.bfloat16, device="cuda")
    cache[1] = 1
    table = torch.zeros(1, PAGES, dtype=torch.int32)
    table[0, -1] = 1
    cache[1, 1, BS - 2, 0, 3] = math.nan  # token 2^31 - 2
    q = torch.ones(news, 1, 16, dtype=torch.bfloat16, device="cuda")
    out, lse = FullCache(cache, "kv_first").attend(
        q, table.cuda(), ints([2 ** 31 - 1]), q_starts=ints([0, news]), max_q=news, return_lse=True)
    assert torch.isnan(out[-1, 0, 3])
    out[-1, 0, 3] = 1
    # Weights are 1: a part's sums are whole numbers, of 2^23 tokens at most, and the join of up to
    # 1,024 parts rounds by 2^-24 each, 2^-14 in all: less than half a step of bf16 (2^-9 below 1).
    assert torch.all(out == 1)
    # the log is off by that, its own rounding (2^-20 of 22 each in two steps) and the missing tokens
    assert torch.all((lse.double() - 31 * math.log(2.0)).abs() <= 2.0 ** -13)
