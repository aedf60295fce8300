"""The weights of tokens on the GPU where a wave, a workgroup or a call takes them in turns: rounds of
tokens, and more query heads on a KV head than share a prefix's tiles."""

import pytest

from tests.test_gpu_full import Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,dtype", [(64, "bf16"), (80, "f16"), (128, "bf16"), (192, "f16")])
@pytest.mark.parametrize("news,shared", [(4, 5), (9, 7), (16, 4), (40, 3)])
@pytest.mark.parametrize("before", [0, 1100])
def test_a_waves_tokens_in_several_rounds(ext, d, dtype, news, shared, before):
    """A bound far below the lengths leaves one workgroup all of a context's rounds: 20 and 63 rows,
    of which each wave has tokens of its own, and 64 and more, which the waves share."""
    Batch("kv_first", 16, 1, shared, d, dtype, [1500], [news], seed=news,
          prefixes=[before] if before else [], groups=[0, 1]).check(max_len=1, prefix_len=1)
