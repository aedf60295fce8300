"""A 4-bit cache on the framework's own path: staged step by step (StepStager) into a store's tables
(StoreTables), restored from them into a spare's caches at other head slots (Restorer), and
attended over there."""

import pytest
import torch

from everserve_amd.state import staging
from everserve_amd.state.fp4 import Fp4Cache
from everserve_amd.state.restore import Restorer
from everserve_amd.state.store import StoreTables
from tests.cases import LAYOUTS

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("d", [64, 72, 128])
def test_a_staged_and_restored_four_bit_cache_gives_the_same_answers(ext, layout, d):
    g = torch.Generator(device="cuda").manual_seed(d)
    n_layers, blocks, bs, heads, shared = 3, 40, 16, 3, 2
    rank = [Fp4Cache.empty(blocks, bs, heads, d, layout) for _ in range(n_layers)]
    names = [f"model.layers.{i}.self_attn.attn" for i in range(n_layers)]
    tables = torch.randperm(blocks, device="cuda", generator=g).int()[:24].reshape(2, 12)
    lens = [0, 0]
    store = StoreTables(ext, blocks * bs)
    with staging.StepStager(ext, dict(zip(names, (c.tensor for c in rank))), [0, 2],
                            store.sink, depth=2) as st:
        # two prompts, then single tokens; a padding id in each step
        for step, new in enumerate([(70, 131), (1, 1), (1, 1), (40, 0), (1, 1)], start=1):
            slots = []
            for s, k in enumerate(new):
                t = torch.arange(lens[s], lens[s] + k, device="cuda")
                slots.append(tables[s][t // bs].long() * bs + t % bs)
                lens[s] += k
            slots = torch.cat(slots + [torch.tensor([-1], device="cuda")])
            for name, c in zip(names, rank):
                x = torch.randn(2, len(slots), heads, d, device="cuda", generator=g).bfloat16()
                c.write(slots, x[0], x[1])
                st.save(name, c.tensor, slots)
            st.commit(epoch=1, step=step, committed_tokens={"r": step})
        st.flush()
    store.flush()

    spare = [Fp4Cache.empty(blocks, bs, 2, d, layout) for _ in range(n_layers)]
    Restorer(ext, [c.tensor for c in spare]).restore(store.restore_tables(), {0: 1, 2: 0})
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = torch.randn(2, heads, shared, d, device="cuda", generator=g).bfloat16()
    moved = q[:, [2, 0]].reshape(2, 2 * shared, d)  # the spare's head slots hold ours 2 and 0
    for a, b in zip(rank, spare):
        want, lse = a.attend(q.reshape(2, heads * shared, d), tables, n, return_lse=True)
        got, got_lse = b.attend(moved, tables, n, return_lse=True)
        assert torch.equal(got.view(2, 2, shared, d), want.view(2, heads, shared, d)[:, [2, 0]])
        assert torch.equal(got_lse.view(2, 2, shared), lse.view(2, heads, shared)[:, [2, 0]])
        assert torch.isfinite(lse).all() and want.abs().sum() > 0
