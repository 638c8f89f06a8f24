"""How the attention of many rows is divided among workgroups: every tile and part is computed once, whatever the requests, on caches in
16 bits and in MXFP4."""
import pytest
import torch

from tests.attention_util import Step, assert_attention
from tests.mxfp4_util import MxStep
from tests.test_attention import attend

HALF, BF16 = torch.float16, torch.bfloat16

# (requests, heads, kv_heads, dim, block_size, dtype, window, sinks)
CASES = {
    "a wave of requests, in parts": ([(700 + 11 * i, 5) for i in range(64)], 8, 1, 64, 16, HALF, 0, 0),
    "more than a wave, in parts": ([(1400 - 9 * i, 5 + i % 3) for i in range(70)], 8, 1, 64, 16, HALF, 0, 0),
    "more than a wave, in parts, some without tokens": ([(900 + i, (i % 4) * 4) for i in range(130)], 8, 1, 128, 16, BF16, 0, 0),
    "more than a wave behind long contexts": ([(60 + 90 * i, 6) for i in range(70)], 8, 1, 64, 64, HALF, 0, 0),
    "more than four waves": ([(40 + i, 5 + i % 7) for i in range(300)], 8, 1, 64, 16, HALF, 0, 0),
    "more tiles than workgroups": ([(64 + 40 * (i % 13), 33) for i in range(40)], 32, 8, 64, 16, BF16, 0, 0),
    "a prompt among requests without tokens": ([(0, 0)] * 5 + [(700, 700)] + [(0, 0)] * 70, 4, 2, 128, 16, HALF, 0, 0),
    "windows of more than a wave": ([(2000 + 17 * i, 6) for i in range(80)], 8, 1, 64, 16, HALF, 600, 5),
    "wide heads, in parts": ([(3000 - 100 * i, 20) for i in range(9)], 8, 2, 256, 16, HALF, 0, 0),
    "wide heads, more tiles than run at once": ([(2300 + 10 * i, 9) for i in range(40)], 64, 8, 256, 64, HALF, 0, 0),
}


@pytest.mark.gpu
@pytest.mark.parametrize("made", [Step, MxStep])
@pytest.mark.parametrize("name", list(CASES))
def test_division(name, made):
    requests, heads, kv_heads, dim, block, dtype, window, sinks = CASES[name]
    s = made(31, requests, heads, kv_heads, dim, block, dtype, "head", window, sinks)
    got = attend(s)
    assert_attention(got, s, name)
    assert torch.equal(got, attend(s)), "a second call on the same inputs differs"
    assert_attention(attend(s, max_context=300), s, f"{name}, contexts longer than the host said")


@pytest.mark.gpu
@pytest.mark.parametrize("made", [Step, MxStep])
def test_division_behind_a_prefix(made):
    requests = [(200 + 9 * i, 5) for i in range(70)]
    s = made(32, requests, 8, 1, 64, 16, HALF, prefix=600)
    assert_attention(attend(s), s, "more requests than a wave behind a prefix")
