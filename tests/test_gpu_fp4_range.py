"""The 4-bit cache over the whole range of its format, and the precision of f16 answers."""

import numpy as np
import pytest
import torch

from everserve_amd.state.fp4 import Fp4Cache
from oracle import fp4
from tests.test_gpu_fp4 import LAYOUTS, TYPES, canonical, check, filled

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


@pytest.mark.parametrize("layout", LAYOUTS)
def test_every_scale_byte_reads_as_its_power_of_two(ext, layout):
    d, bs = 64, 16
    host = np.zeros((256, 2, 2, fp4.row_bytes(d)), dtype=np.uint8)  # [slot, head, K or V, byte]
    pairs = np.arange(16) | (np.arange(16) << 4)
    host[..., :d // 2] = np.concatenate((pairs, pairs[::-1]))  # every code in each group
    host[..., d // 2] = np.arange(256)[:, None, None]
    host[..., d // 2 + 1] = np.arange(256)[::-1, None, None]
    cache = Fp4Cache.empty(16, bs, 2, d, layout)
    cache.tensor.copy_(torch.from_numpy(_as(layout, host, bs)))
    assert np.array_equal(canonical(cache).reshape(host.shape), host)
    for dtype in TYPES.values():
        rows = cache.read(torch.arange(256, device="cuda"), dtype)
        for kv in (0, 1):
            want = torch.from_numpy(fp4.decode(host[:, :, kv], d)).to(dtype)
            assert torch.equal(torch.isnan(rows[kv].cpu()), torch.isnan(want))
            assert torch.equal(torch.nan_to_num(rows[kv].cpu(), 7, None, None),
                               torch.nan_to_num(want, 7, None, None))


def _as(layout, rows, bs):
    """[slots, heads, 2, bytes] as the tensor of a cache."""
    n, heads, _, half = rows.shape
    x = rows.reshape(n // bs, bs, heads, 2, half)
    order = {"kv_first": (3, 0, 1, 2, 4), "blocks_first": (0, 3, 1, 2, 4),
             "combined": (0, 2, 1, 3, 4)}[layout]
    x = x.transpose(order)
    return np.ascontiguousarray(x.reshape(*x.shape[:3], 2 * half) if layout == "combined" else x)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_rows_below_the_least_scale_are_rounded_like_others(ext, dtype):
    # from the smallest values there are, each a number of steps of 2^-149, up to 2^-120
    g = np.random.default_rng(3)
    x = g.standard_normal((90, 2, 64)) * np.exp2(g.integers(-150, -120, (90, 2, 1)))
    x = torch.from_numpy(x).to(TYPES[dtype])
    cache = Fp4Cache.empty(9, 10, 2, 64)
    cache.write(torch.arange(90, device="cuda"), x.cuda(), -x.cuda())
    got = canonical(cache).reshape(90, 2, 2, -1)
    assert np.array_equal(got[:, :, 0], fp4.encode(x.double().numpy()))
    assert np.array_equal(got[:, :, 1], fp4.encode(-x.double().numpy()))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("byte", [0, 1, 3])
@pytest.mark.parametrize("news", [1, 90])
def test_values_with_the_least_scales_keep_their_bits(ext, dtype, byte, news):
    """Every V has the same small scale: the answers are those with the scale 2^0 times a power of
    two, to the output's own rounding (f32 keeps 2^-149, a weighted mean loses a few of those)."""
    d, n = 64, 150
    cache, tables = filled("kv_first", 16, 2, d, [n], 6)
    q = torch.randn(news, 8, d, generator=torch.Generator().manual_seed(3)).to(TYPES[dtype]).cuda()
    how = dict(q_starts=torch.tensor([0, news]).int().cuda(), max_q=news)
    lens = torch.tensor([n]).int().cuda()
    values = cache.tensor[1]
    outs = []
    for b in (127, byte):
        values[..., d // 2:d // 2 + 2] = b
        outs.append(cache.attend(q, tables.cuda(), lens, **how).double())
    scale = 2.0 ** (byte - 127)
    steps = {"bf16": 2.0 ** -133, "f16": 2.0 ** -24}[dtype]  # below the normals
    room = outs[0].abs() * scale * torch.finfo(TYPES[dtype]).eps + steps + n * 2.0 ** -148
    assert torch.all((outs[1] - outs[0] * scale).abs() <= room)


@pytest.mark.parametrize("d,news,lens", [(64, 1, [500, 90]), (80, 40, [300]), (128, 1, [3000, 7]),
                                         (128, 9, [700, 40]), (200, 100, [260]), (256, 1, [65])])
@pytest.mark.parametrize("layout", LAYOUTS)
def test_f16_answers_round_their_weights_to_sixteen_bits(ext, layout, d, news, lens):
    """For f16 queries a weight is the sum of two bf16: off by 2^-17 of itself at most (half a step
    of the second, which holds what the first left, at most 2^-8 of the weight). The answers are as
    near as that and their own rounding allow, eight times as near as one bf16 would be."""
    cache, tables = filled(layout, 16, 2, d, lens, d)
    g = torch.Generator().manual_seed(news)
    q = torch.randn(news * len(lens), 6, d, generator=g).half().cuda()
    starts = np.arange(0, news * len(lens) + 1, news)
    out, lse = cache.attend(q, tables.cuda(), torch.tensor(lens).int().cuda(), return_lse=True,
                            q_starts=torch.from_numpy(starts).int().cuda(), max_q=news)
    check(cache, q, tables, lens, starts, d ** -0.5, out, lse)
    want, _, reach, worst = fp4.attend(q.double().cpu().numpy(), canonical(cache), d,
                                       tables.numpy(), lens, starts, d ** -0.5)
    n = max(lens) + 16
    # scores, exponentials and sums as `check` has them
    score = (d + 4) * 2.0 ** -24 * worst + 2.0 ** -22 * worst + 2.0 ** -22
    weight = (2 * score + 2 * n * 2.0 ** -24)[..., None]
    room = reach * (weight + 2.0 ** -16 * (1 + weight))
    room += (np.abs(want) + room) * 2.0 ** -11 + 2.0 ** -25  # and half a step below the normals
    off = np.abs(out.double().cpu().numpy() - want)
    assert np.all(off <= room), float((off / room).max())
