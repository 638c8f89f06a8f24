"""The order in which the tiles and parts of a step are dealt: tiles that all have as many parts, and tiles that do not."""
import ctypes

import pytest
import torch

from autogptq.tvm_amd import _lib
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
    "few long lists among short ones, wide heads": ([(6300, 300), (298, 298), (72, 72), (1000, 17), (122, 4)], 32, 8, 256, 24, BF16, 0, 0),
    "few long lists among short ones": ([(9000, 200)] + [(130 + i, 129) for i in range(20)], 32, 8, 128, 16, HALF, 0, 0),
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
@pytest.mark.parametrize("request_, window, prefix", [((0, 0), 0, 0), ((900, 0), 0, 0), ((40, 40), 0, 0), ((2500, 70), 0, 0), ((2500, 70), 300, 0), ((3, 50), 0, 0),
                                                      ((700, 60), 0, 2500)])
@pytest.mark.parametrize("ahead, behind", [(0, 0), (0, 90), (7, 61)])
def test_one_request(made, request_, window, prefix, ahead, behind):
    """Alone in its step, with or without tokens, some of them before its context, in a step that is padded."""
    s = made(43, [request_], 8, 2, 64, 16, HALF, "head", window, 3 if window else 0, prefix)
    want, size = s.expected()
    n = s.tokens
    nan = lambda rows: torch.full((rows, 8, 64), float("nan"), device="cuda").half()
    s.q = torch.cat([nan(ahead), s.q, nan(behind)])
    s.starts = s.starts + ahead
    nan(len(s.q))      # what the result's memory holds
    got = attend(s)
    assert bool((got[:ahead] == 0).all()) and bool((got[ahead + n:] == 0).all())
    assert bool(((got[ahead:ahead + n].double() - want).abs() <= 2.25 * 2.0 ** -11 * size + 2.0 ** -24).all())


@pytest.mark.gpu
@pytest.mark.parametrize("made", [Step, MxStep])
def test_lengths_that_the_host_did_not_expect(made):
    """Contexts behind the longest that the host knows: longer parts, as many for every tile."""
    s = made(42, [(3000, 40), (2900, 40), (2950, 33)], 8, 2, 64, 16)
    for hint in (600, 1500, 100000):
        assert_attention(attend(s, max_context=hint), s, f"max_context={hint}")


def mx_workspace(tokens, requests, context, heads, kv_heads, dim, window=0, sinks=0, prefix=0):
    """Bytes that a call over a cache in MXFP4 needs (blocks of 16 tokens, a table as wide as the context)."""
    p = 0x1000
    groups, scale = -(-dim // 32), 2 if dim <= 64 else 4 if dim <= 128 else 8
    cache = _lib.CacheMx(k=p, v=p, k_scales=p, v_scales=p, type=0, blocks=1000, block_size=16, heads=kv_heads, dim=dim,
                         block_stride=256 * groups * kv_heads, slot_stride=16 * groups, head_stride=256 * groups,
                         scale_block_stride=16 * scale * kv_heads, scale_slot_stride=scale, scale_head_stride=16 * scale)
    a = _lib.Attention()
    a.q = a.out = a.tables = a.starts = a.contexts = a.prefix_blocks = p
    a.tokens, a.requests, a.heads, a.max_context, a.scale = tokens, requests, heads, context, 0.1
    a.window, a.sinks, a.prefix_length = window, sinks, prefix
    a.table_width = a.table_stride = -(-context // 16)
    a.q_token_stride, a.q_head_stride = heads * dim, dim
    return _lib.lib().gptq_hip_attention_mx_workspace_bytes(ctypes.byref(cache), ctypes.byref(a))


def size_of(rows, dim):
    """... that the parts of so many rows take: counters, two statistics and dim values a row."""
    return 65536 + -(-rows * 8 // 256) * 256 + rows * dim * 4


@pytest.mark.parametrize("requests, context, kv_heads, dim, units", [
    (1, 128, 8, 128, 1), (1, 200, 8, 128, 1), (1, 256, 8, 128, 1), (16, 256, 8, 128, 1),       # one of 256: no parts to join
    (1, 257, 8, 128, 3), (1, 512, 8, 128, 4), (1, 768, 8, 128, 6), (1, 1024, 8, 128, 8), (4, 1024, 8, 64, 8), (3, 700, 2, 256, 6),
    (8, 512, 8, 128, 4), (1, 1025, 8, 128, 5), (1, 2048, 8, 128, 8),
    (8, 520, 8, 128, 3), (16, 300, 8, 128, 2), (33, 129, 8, 128, 1)])                          # more than a CU each
def test_units_of_short_contexts(requests, context, kv_heads, dim, units):
    """A single token's keys are dealt in units of 128 where those are up to eight, more than one of 256, and have a CU each; else of 256."""
    tiles = requests * 4 // 16 + requests
    rows = 2 * min(256 * (2 if dim > 128 else 4) // kv_heads, tiles * units) * kv_heads * 16
    assert mx_workspace(requests, requests, context, 4 * kv_heads, kv_heads, dim) == size_of(rows, dim)
