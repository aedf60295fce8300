"""Attention calls with queries and nothing to do for them: every row that comes back is one that
sees nothing, whatever the memory held before."""

import math

import pytest
import torch

from tests.test_gpu_fp4 import filled

pytestmark = pytest.mark.gpu


def soil(*shapes):
    """Leave memory of these f32 shapes behind, for the next tensors, that is no number."""
    held = [torch.full(s, math.nan, device="cuda") for s in shapes]
    torch.cuda.synchronize()
    del held


@pytest.mark.parametrize("how", ["no sequence", "no query"])
@pytest.mark.parametrize("tokens", [1, 70])
def test_rows_without_work_are_zeros(ext, how, tokens):
    cache, tables = filled("kv_first", 16, 2, 64, [40, 7], 3)
    tables, lens = tables.cuda(), torch.tensor([40, 7], dtype=torch.int32, device="cuda")
    starts = torch.zeros(3, dtype=torch.int32, device="cuda")
    max_q = 0 if how == "no query" else 5
    if how == "no sequence":
        tables, lens, starts = tables[:0], lens[:0], starts[:1]
    q = torch.randn(tokens, 8, 64, device="cuda").bfloat16()
    for _ in range(3):
        soil((tokens, 4, 64), (tokens, 8))
        out, lse = cache.attend(q, tables, lens, q_starts=starts, max_q=max_q, return_lse=True)
        assert torch.all(out == 0) and torch.all(lse == -math.inf)
    given = torch.full_like(q, 7.0)  # a caller's own rows are theirs: nothing names them
    assert cache.attend(q, tables, lens, q_starts=starts, max_q=max_q, out=given) is given
    assert torch.all(given == 7)
