"""``PagedCache(quantize="mxfp4")``, and ``PagedCache.read`` of both kinds."""
import os
import sys

import pytest
import torch

from autogptq.tvm_amd import PagedCache
from autogptq.tvm_amd.attention import Mxfp4
from tests.mxfp4_util import decode, encode

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HALF, BF16 = torch.float16, torch.bfloat16


def cache(**more):
    return PagedCache(**{**dict(layers=2, blocks=40, block_size=8, kv_heads=2, dim=64, max_requests=4, max_context=160, quantize="mxfp4"), **more})


def draw(gen, n, heads=2, dim=64, dtype=HALF):
    return torch.randn(2, n, heads, dim, generator=gen).to(dtype).cuda()


@pytest.mark.gpu
def test_a_decoder_is_served_from_it():
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    try:
        import serve_paged
    finally:
        sys.path.pop(0)
    # (every layer's attention against a plain one over what the cache gives back: the shares and the result are rounded to fp16, 2^-11 each
    # of sums that are a few times the result; the example asserts 2e-2 at every step)
    assert serve_paged.main(verbose=False, quantize="mxfp4") < 2e-2


def test_refusals():
    for more in (dict(quantize="int4"), dict(quantize="mxfp4", dtype=torch.float32), dict(dim=60)):
        with pytest.raises(ValueError):
            cache(device="cpu", **more)
    c = cache(device="cpu")
    assert isinstance(c.k[1], Mxfp4) and c.k[0].codes.shape == (40, 8, 2, 32) and c.v[1].scales.shape == (40, 8, 2, 2)
    x = torch.zeros(3, 2, 64)
    for call in (lambda: c.write(0, x.half(), x.bfloat16(), None), lambda: c.write(0, x, x, None), lambda: c.attend(0, x.bfloat16(), None)):
        with pytest.raises(ValueError, match="holds values of torch.float16"):
            call()
    # (rows of 80 values and of 96 take the same bytes)
    c = cache(device="cpu", dim=80)
    for x in (torch.zeros(3, 2, 96).half(), torch.zeros(3, 2, 72).half()):
        for call in (lambda: c.write(0, x, x, None), lambda: c.attend(0, x, None)):
            with pytest.raises(ValueError, match="80 of a head"):
                call()
    with pytest.raises(IndexError):
        c.read(0, 4)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        c.read(0, 1)


@pytest.mark.gpu
@pytest.mark.parametrize("quantize, dtype, dim", [("mxfp4", HALF, 64), ("mxfp4", BF16, 80), (None, BF16, 80), (None, HALF, 64)])
def test_read(quantize, dtype, dim):
    gen = torch.Generator().manual_seed(2)
    c = cache(quantize=quantize, dtype=dtype, dim=dim)
    seen = {r: [] for r in range(4)}
    for requests, counts in (((0, 2), (30, 9)), ((2, 1, 0), (1, 20, 1)), ((1,), (7,))):
        s = c.step(requests, counts)
        for layer in (0, 1):
            k, v = draw(gen, sum(counts), dim=dim, dtype=dtype)
            c.write(layer, k, v, s)
            for i, r in enumerate(requests):
                at = slice(int(s.starts[i]), int(s.starts[i + 1]))
                seen[r].append((layer, k[at], v[at]))
    for r in range(4):
        for layer in (0, 1):
            for i, got in enumerate(c.read(layer, r)):
                parts = [x[1 + i] for x in seen[r] if x[0] == layer]
                want = torch.cat(parts) if parts else torch.empty(0, 2, dim, dtype=dtype, device="cuda")
                assert got.dtype == dtype and got.shape == want.shape
                assert torch.equal(got.double(), decode(*encode(want), dim)) if quantize else torch.equal(got, want)
    assert c.trim(0, window=6, sinks=3) == 2            # blocks 1 and 2 of 4
    k, _ = c.read(1, 0)
    want = [x[1] for x in seen[0] if x[0] == 1]
    want = decode(*encode(torch.cat(want)), dim) if quantize else torch.cat(want).double()
    want[8:24] = 0
    assert torch.equal(k.double(), want)


@pytest.mark.gpu
def test_a_run_of_them():
    """Prompts, decoding, requests behind a prefix and a window with blocks given back: the same as over what was read back."""
    gen = torch.Generator().manual_seed(4)
    c, plain = cache(), cache(quantize=None)
    def go(requests, counts, **mask):
        n = sum(counts)
        k, v = draw(gen, n)
        q = torch.randn(n, 4, 64, generator=gen).half().cuda()
        steps = [x.step(requests, counts) for x in (c, plain)]
        c.write(1, k, v, steps[0])
        k, v = (decode(*encode(x), 64).half() for x in (k, v))
        plain.write(1, k, v, steps[1])
        got, want = (x.attend(1, q, s, **mask).double() for x, s in zip((c, plain), steps))
        # both round the shares and the result once; values are below 8
        assert bool(((got - want).abs() <= 4.5 * 2.0 ** -11 * 8).all())
        return got
    go([3], [1], window=20, sinks=2)        # (tables that differ from the order of requests)
    go([0], [30])
    for x in (c, plain):
        x.share(0, 1), x.share(0, 2)
    go([1, 2], [5, 1])
    for _ in range(3):
        go([1, 2], [1, 1])
    go([3], [70], window=20, sinks=2)
    for _ in range(3):
        assert c.trim(3, 20, 2) == plain.trim(3, 20, 2)
        go([3], [3], window=20, sinks=2)
    for x in (c, plain):
        for r in (1, 2, 0, 3):
            x.free(r)
        assert x.free_blocks == 40
