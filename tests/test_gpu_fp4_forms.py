"""Forms of the calls' arguments that a program may hand over: queries on any element, tables that are
views, and lists that take several launches."""

import numpy as np
import pytest
import torch

from everserve_amd.state.fp4 import Fp4Cache
from everserve_amd.state.pages import PageMover
from oracle import fp4
from tests.test_gpu_fp4 import LAYOUTS, TYPES, canonical, check, filled

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("news", [1, 3, 50])
def test_queries_on_any_element_and_tables_that_are_views(ext, layout, dtype, news):
    d, lens = 72, [150, 33, 70]
    cache, tables = filled(layout, 16, 2, d, lens, news)
    g = torch.Generator().manual_seed(news)
    wide = torch.randn(3 * news, 2 * 4 + 1, d + 3, generator=g).to(TYPES[dtype]).cuda()
    q = wide[:, 1:, 1:1 + d]  # a token, a head and the first element off 16 bytes
    assert q.data_ptr() % 16 and not q.is_contiguous()
    apart = torch.full((5, tables.shape[1] + 7), -9, dtype=torch.int32)
    apart[1:4, 2:2 + tables.shape[1]] = tables
    view = apart.cuda()[1:4, 2:2 + tables.shape[1]]
    starts = np.arange(0, 3 * news + 1, news)
    out, lse = cache.attend(q, view, torch.tensor(lens).int().cuda(), max_q=news, return_lse=True,
                            q_starts=torch.from_numpy(starts).int().cuda())
    check(cache, q, tables, lens, starts, d ** -0.5, out, lse)
    plain = cache.attend(q.contiguous(), tables.cuda(), torch.tensor(lens).int().cuda(),
                         q_starts=torch.from_numpy(starts).int().cuda(), max_q=news)
    assert torch.equal(out, plain)


def test_sequences_may_share_one_table(ext):
    # four sequences at different lengths of one context: a table of stride 0
    cache, tables = filled("combined", 16, 2, 64, [300], 2)
    q = torch.randn(4, 8, 64, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    lens = [300, 17, 0, 256]
    one = tables.cuda().expand(4, -1)
    out = cache.attend(q, one, torch.tensor(lens).int().cuda())
    check(cache, q, tables.expand(4, -1), lens, np.arange(5), 64 ** -0.5, out, None)


def test_rows_that_take_several_launches(ext):
    # a launch takes 2^28 pieces of rows: here 65,536 rows of 512 heads of 256 written, 256 of
    # 32,768 heads of 256 read
    cache = Fp4Cache.empty(2, 4, 512, 256)
    n = (1 << 16) + 5
    slots = torch.full((n,), -1, device="cuda")
    slots[torch.tensor([0, 65535, 65536, n - 1])] = torch.tensor([0, 3, 5, 7], device="cuda")
    x = torch.randn(2, 1, 512, 256, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    x = x.bfloat16()
    cache.write(slots, x[0].expand(n, -1, -1), x[1].expand(n, -1, -1))
    got = canonical(cache).reshape(8, 512, 2, -1)
    for kv in (0, 1):
        want = fp4.encode(x[kv, 0].double().cpu().numpy())
        for s in range(8):
            assert np.array_equal(got[s, :, kv], want if s in (0, 3, 5, 7) else np.zeros_like(want))

    cache = Fp4Cache.empty(1, 4, 32768, 256)
    x = torch.randn(1, 32768, 2, 256, device="cuda").bfloat16()
    cache.write(torch.tensor([2], device="cuda"), x[:, :, 0], x[:, :, 1])
    want = cache.read(torch.tensor([2], device="cuda"), torch.bfloat16)
    n = 256 + 3
    slots = torch.full((n,), -1, device="cuda")
    slots[255:257], slots[n - 1] = 2, 2
    got = cache.read(slots, torch.bfloat16)
    for a, b in zip(got, want):
        for i in (255, 256, n - 1):
            assert torch.equal(a[i], b[0])
        assert not a[:255].any() and not a[257:n - 1].any()


def test_page_copies_that_take_several_launches(ext):
    # pages of 65,536 words of a byte: a launch takes 32,767 pairs
    layer = torch.randint(0, 256, (5, 2, 128, 4, 65), dtype=torch.uint8, device="cuda")[..., :64]
    want = layer.clone()
    n = 32767 + 9
    src = torch.full((n,), -1, dtype=torch.int32, device="cuda")
    dst = torch.full((n,), -1, dtype=torch.int32, device="cuda")
    src[0], dst[0] = 1, 0
    src[32766], dst[32766] = 2, 3
    src[n - 1], dst[n - 1] = 1, 4
    mover = PageMover([layer], "blocks_first")
    mover.copy(src, dst)
    want[0], want[3], want[4] = want[1].clone(), want[2].clone(), want[1].clone()
    assert torch.equal(layer, want)
    with pytest.raises(RuntimeError, match="device count"):
        mover.copy(src, dst, torch.tensor([1], dtype=torch.int32, device="cuda"))
