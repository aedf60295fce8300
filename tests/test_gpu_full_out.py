"""Where attention over full-width pages writes: beside the queries, and never among them."""

import pytest
import torch

from tests.test_gpu_full import Batch, ints

pytestmark = pytest.mark.gpu


def test_outputs_beside_and_between_the_queries(ext):
    b = Batch("kv_first", 16, 2, 2, 64, "bf16", [70, 33, 5], [1] * 3, prefixes=[40], groups=[0, 2])
    want = b.attend()[0]
    n = want.numel()
    # one tensor for both, one behind the other; queries that lie apart, the output in a gap of them
    for wide, first in ((256, n), (256, 0), (2048, 256), (2048, 2048 + 512)):
        buf = torch.zeros(8 * 2048, dtype=torch.bfloat16, device="cuda")
        at = n if first == 0 else 0
        q = buf[at:at + 3 * wide].view(3, wide)[:, :256].view(3, 4, 64)
        q.copy_(b.q)
        out = buf[first:first + n].view(3, 4, 64)
        got = b.cache.attend(q, b.tables.cuda(), ints(b.lens), prefix=b.prefix(), out=out)
        assert got is out and torch.equal(out, want)


def test_an_output_that_overlaps_the_queries_is_refused(ext):
    b = Batch("kv_first", 16, 2, 2, 64, "bf16", [70, 33, 5], [1] * 3)
    buf = torch.zeros(8 * 2048, dtype=torch.bfloat16, device="cuda")
    q = buf[:3 * 256].view(3, 4, 64)
    for first in (0, 8, 256, 3 * 256 - 8):
        out = buf[first:first + 3 * 256].view(3, 4, 64)
        with pytest.raises(RuntimeError, match="must not be the queries"):
            b.cache.attend(q, b.tables.cuda(), ints(b.lens), out=out)
    fused = buf[:3 * 1024].view(3, 1024)[:, :256].view(3, 4, 64)
    with pytest.raises(RuntimeError, match="must not be the queries"):  # reaches into the next token
        b.cache.attend(fused, b.tables.cuda(), ints(b.lens), out=buf[512:512 + 768].view(3, 4, 64))

