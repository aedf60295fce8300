"""The 4-bit cache over the whole range of its format."""

import pytest
import torch

from tests.test_gpu_fp4 import TYPES, filled

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("byte", [253, 254])
@pytest.mark.parametrize("d", [64, 128, 200])
@pytest.mark.parametrize("news,shared", [(3, 4), (16, 1), (100, 2)])
@pytest.mark.parametrize("back", [0, 2])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_values_past_the_largest_number_reach_only_the_rows_that_see_them(ext, byte, d, news,
                                                                          shared, back, dtype):
    """A token whose V has a group of infinite values (4 times 2^126 is no finite f32), at the last
    places of a chunk: the rows before it are as without it, bit for bit."""
    n = 200
    cache, tables = filled("kv_first", 16, 1, d, [n, n], 6)
    at = n - 1 - back
    page, off, grp = int(tables[0, at // 16]), at % 16, 1
    how = dict(q_starts=torch.tensor([0, news, 2 * news]).int().cuda(), max_q=news)
    q = torch.randn(2 * news, shared, d, generator=torch.Generator().manual_seed(3))
    q = q.to(TYPES[dtype]).cuda()
    lens = torch.tensor([n, n], device="cuda").int()
    want = cache.attend(q, tables.cuda(), lens, **how)
    hit = max(news - 1 - back, 0)  # the first query that sees the token
    for kv in (1, 0):
        row = cache.tensor[kv, page, off, 0]
        kept = row.clone()
        row[16 * grp:16 * grp + 16] = 0x76  # 4 and 6 steps
        row[d // 2 + grp] = byte
        out = cache.attend(q, tables.cuda(), lens, **how)
        row.copy_(kept)
        assert torch.equal(out[:hit], want[:hit]) and torch.equal(out[news:], want[news:])
        seen, group = out[hit:news], slice(32 * grp, 32 * grp + 32)
        if kv == 1:
            assert torch.all(seen[..., group] == torch.inf)
            other = torch.ones(d, dtype=torch.bool, device="cuda")
            other[group] = False
            assert torch.equal(seen[..., other], want[hit:news][..., other])
