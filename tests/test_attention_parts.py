"""The order in which the tiles and parts of a step are dealt: tiles that all have as many parts, and tiles that do not."""
import pytest
import torch

from tests.attention_util import Step, assert_attention
from tests.mxfp4_util import MxStep
from tests.test_attention import attend

HALF, BF16 = torch.float16, torch.bfloat16

# (requests, heads, kv_heads, dim, block_size, dtype, window, sinks)
CASES = {
    "five parts each": ([(1064, 64)] * 4, 32, 8, 64, 16, HALF, 0, 0),
    "five parts each, wide heads": ([(1064, 64)] * 4, 8, 2, 256, 16, BF16, 0, 0),
    "as many parts among requests without tokens": ([(0, 0), (2100, 30), (5, 0), (2090, 77), (2080, 9), (900, 0)], 8, 2, 128, 16, HALF, 0, 0),
    "one request": ([(3000, 100)], 4, 1, 128, 24, BF16, 0, 0),
    "one request more than a wave ends with": ([(0, 0)] * 63 + [(2000, 70)], 8, 2, 64, 16, HALF, 0, 0),
    "two parts each, more than run at once": ([(2000 - 11 * (i % 7), 9) for i in range(38)], 32, 8, 64, 64, HALF, 0, 0),
    "one request of fewer parts": ([(2100, 30)] * 5 + [(200, 30)], 8, 2, 64, 16, HALF, 0, 0),
    "as many parts under a window": ([(4000 + 100 * i, 40) for i in range(6)], 8, 2, 128, 16, BF16, 900, 4),
    "no part is seen": ([(0, 5)] * 7 + [(0, 0)], 8, 2, 64, 16, HALF, 0, 0),
}


@pytest.mark.gpu
@pytest.mark.parametrize("made", [Step, MxStep])
@pytest.mark.parametrize("name", list(CASES))
def test_parts(name, made):
    requests, heads, kv_heads, dim, block, dtype, window, sinks = CASES[name]
    s = made(41, requests, heads, kv_heads, dim, block, dtype, "head", window, sinks)
    hint = 3000 if not s.most else s.most
    got = attend(s, max_context=hint)
    assert_attention(got, s, name)
    assert torch.equal(got, attend(s, max_context=hint)), "a second call on the same inputs differs"


@pytest.mark.gpu
@pytest.mark.parametrize("made", [Step, MxStep])
def test_lengths_that_the_host_did_not_expect(made):
    """Contexts behind the longest that the host knows: longer parts, as many for every tile."""
    s = made(42, [(3000, 40), (2900, 40), (2950, 33)], 8, 2, 64, 16)
    for hint in (600, 1500, 100000):
        assert_attention(attend(s, max_context=hint), s, f"max_context={hint}")
