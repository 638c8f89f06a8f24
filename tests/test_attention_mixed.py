"""Batches over a cache in MXFP4 whose requests of few rows have a launch of the few-rows kernel and whose others the kernel of tiles:
that they are divided so, and what both launches share (the workspace, the tokens of no request, a captured graph)."""
import copy
import functools
from types import SimpleNamespace

import pytest
import torch

from tests.attention_util import ROUNDING, assert_attention
from tests.mxfp4_util import MxStep
from tests.test_attention import attend, captured, overwrite
from tests.test_attention_parts import mx_workspace, size_of

HALF, BF16 = torch.float16, torch.bfloat16


def singles(n, top, step):
    return [(1 + (top - 1 - step * i) % top, 1) for i in range(n)]


# (requests, heads, kv_heads, dim, block_size, dtype, window, sinks), rows of a few-rows tile, and workgroups of it that a CU holds
CASES = {
    "dim 64": (singles(64, 5000, 397) + [(3000, 700), (900, 400), (0, 0), (2000, 4), (2000, 5)], 16, 4, 64, 16, HALF, 0, 0, 16, 4),
    "dim 128": (singles(66, 4000, 211) + [(4000, 4), (3900, 900), (700, 5), (0, 0), (300, 300)], 16, 4, 128, 64, BF16, 0, 0, 16, 4),
    "dim 80, window": (singles(90, 4100, 97) + [(4000, 500), (4100, 2), (3000, 3), (200, 200)], 21, 3, 80, 24, HALF, 2500, 5, 16, 4),
    "dim 256": (singles(62, 2000, 97) + [(1500, 500), (700, 700), (0, 0), (1000, 8), (1000, 9)], 16, 8, 256, 16, HALF, 0, 0, 16, 2),
    "two operands, dim 64": (singles(62, 3000, 131) + [(3000, 300), (0, 0), (700, 2), (40, 40)], 96, 4, 64, 16, BF16, 0, 0, 32, 3),
    "two operands, dim 128": (singles(62, 3000, 131) + [(3000, 300), (0, 0), (700, 2), (40, 40)], 96, 4, 128, 16, HALF, 0, 0, 32, 2),
    "a piece among requests that are empty": ([(3000, 1)] * 30 + [(0, 0)] * 39 + [(3000, 600)], 16, 4, 64, 16, HALF, 0, 0, 16, 4),
}


@functools.lru_cache(maxsize=2)
def made(name, seed):
    requests, heads, kv_heads, dim, block, dtype, window, sinks, rows, resident = CASES[name]
    s = MxStep(seed, requests, heads, kv_heads, dim, block, dtype, "head", window, sinks)
    return s, s.expected()


def step(name, seed=51):
    """A step of its own, on tensors that others may share; what is expected of it as it is, is worked out once."""
    s, expected = made(name, seed)
    s = copy.copy(s)
    s.expected = lambda scale=None: expected
    in_two_launches(s, name)
    return s


def in_two_launches(s, name):
    """The tiles of these batches are not divided, so that they need no workspace: what is asked for holds the parts of the
    few-rows launch, two for each of the workgroups that run at once.  More rows a request than the few-rows kernel takes,
    so that it is not the only one."""
    rows, resident = CASES[name][-2:]
    group = s.heads // s.kv_heads
    assert s.tokens * group > (16 if s.dim > 128 else 32) * len(s.requests)
    assert any(0 < n * group <= rows for _, n in s.requests) and any(n * group > rows for _, n in s.requests)
    parts = 2 * (256 * resident // s.kv_heads) * s.kv_heads * rows
    asked = mx_workspace(s.tokens, len(s.requests), s.most, s.heads, s.kv_heads, s.dim, s.window, s.sinks)
    assert asked == size_of(parts, s.dim), f"{name}: not divided into two launches, or in parts"


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(CASES))
def test_mixed(name):
    s = step(name)
    got = attend(s)
    assert_attention(got, s, name)
    for _ in range(3):
        assert torch.equal(got, attend(s)), "a later call on the same inputs differs"


@pytest.mark.gpu
@pytest.mark.parametrize("hint", [0, 1, 300, 7000, 100000])
@pytest.mark.parametrize("name", ["dim 64", "dim 256", "two operands, dim 128"])
def test_max_context_is_a_hint(name, hint):
    """(Also of another division: below the bound no launch for few rows, from 6144 on parts by the lengths.)"""
    s = step(name)
    assert_attention(attend(s, max_context=hint), s, f"{name}, max_context={hint}")


@pytest.mark.gpu
@pytest.mark.parametrize("ahead, behind", [(0, 300), (3, 5), (40, 0)])
@pytest.mark.parametrize("name", ["dim 128", "dim 256", "two operands, dim 64"])
def test_tokens_of_no_request_get_zeros(name, ahead, behind):
    s = step(name)
    want, size = s.expected()
    n = s.tokens
    nan = lambda rows: torch.full((rows, s.heads, s.dim), float("nan"), device="cuda", dtype=s.dtype)
    s.q = torch.cat([nan(ahead), s.q, nan(behind)])
    s.starts = s.starts + ahead
    s.tokens = len(s.q)
    in_two_launches(s, name)
    nan(s.tokens)      # what the result's memory holds
    got = attend(s)
    assert bool((got[:ahead] == 0).all()) and bool((got[ahead + n:] == 0).all())
    assert bool(((got[ahead:ahead + n].double() - want).abs() <= 2.25 * ROUNDING[s.dtype] * size + 2.0 ** -24).all())


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["dim 64", "dim 256", "two operands, dim 128"])
def test_captured_in_a_graph(name):
    """Replays with eager calls of another size, on the same stream, between them."""
    s, other = step(name), step("dim 128", 52)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want, other_want = attend(s), attend(other)
        graph, got = captured(side, lambda: attend(s))
        for _ in range(4):
            got.zero_()
            junk = overwrite()
            graph.replay()
            side.synchronize()
            assert torch.equal(got, want)
            assert all(bool((j == 0x7f).all()) for j in junk), "a replay wrote into another tensor"
            assert torch.equal(attend(other), other_want) and torch.equal(attend(s), want)
            side.synchronize()


@pytest.mark.gpu
def test_captured_with_other_lengths():
    """The lengths of a replay are what the tensors say: requests change launches."""
    s = step("dim 64")
    del s.expected
    s.starts = s.starts.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        attend(s)
        graph, got = captured(side, lambda: attend(s))
        first = s.starts.clone()
        counts = [n for _, n in s.requests]
        for order in (1, 2):
            # some tokens of the piece of 700 (request 64) belong to single requests before it: rows of others, fewer keys
            moved = list(counts)
            for b in range(0, 10 * order):
                moved[b] = min(s.requests[b][0], 1 + 3 * (b % order + 1))
            moved[64] -= sum(moved) - sum(counts)
            s.starts.copy_(torch.cat([torch.zeros(1), torch.tensor(moved).cumsum(0)]).to(first.dtype))
            s.requests = [(c, n) for (c, _), n in zip(s.requests, moved)]
            graph.replay()
            side.synchronize()
            assert_attention(got, s, f"lengths {order}")
            assert torch.equal(got, attend(s))


@pytest.mark.parametrize("name", list(CASES))
def test_the_host_divides_them_so(name):
    requests, heads, kv_heads, dim, _, _, window, sinks = CASES[name][:8]
    in_two_launches(SimpleNamespace(requests=requests, heads=heads, kv_heads=kv_heads, dim=dim, window=window, sinks=sinks,
                                    tokens=sum(n for _, n in requests), most=max(c for c, _ in requests)), name)
