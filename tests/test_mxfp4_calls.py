"""Calls of the cache operators that other files leave out: function transforms, reads far into a cache of 16 bits, the size of an error."""
import pytest
import torch

from autogptq.tvm_amd import attention
from tests.mxfp4_util import MxStep, empty
from tests.test_attention import attend

HALF, BF16 = torch.float16, torch.bfloat16


@pytest.mark.gpu
@pytest.mark.parametrize("prefix", [0, 30])
def test_function_transforms_see_the_attention(prefix):
    from torch.fx.experimental.proxy_tensor import make_fx

    s = MxStep(61, [(40, 1), (30, 20)], 4, 2, 64, 16, prefix=prefix)

    def run(q):
        s.q = q
        return attend(s)
    qs = torch.stack([s.q, s.q * 0.5, s.q.flip(0)])
    got = torch.func.vmap(run)(qs)
    assert got.shape == qs.shape
    for g, q in zip(got, qs):
        assert torch.equal(g, run(q))
    graph = make_fx(run)(qs[0])
    name = "shared_prefix_attention_mx" if prefix else "paged_attention_mx"
    assert any(name in str(n.target) for n in graph.graph.nodes)
    assert torch.equal(graph(qs[1]), run(qs[1]))


@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [True, False])
def test_function_transforms_see_the_read(quantised):
    from torch.fx.experimental.proxy_tensor import make_fx

    slots = torch.tensor([[0, 9, -1, 63], [5, 5, 64, 1], [2, 3, 4, 7]], dtype=torch.int32, device="cuda")
    if quantised:
        cache = empty(4, 16, 2, 64)
        k, v = torch.randn(2, 64, 2, 64, device="cuda").half()
        attention.cache_write(k, v, *cache, torch.arange(64, dtype=torch.int32, device="cuda"))
    else:
        cache = torch.randn(2, 4, 16, 2, 64, device="cuda").half().unbind()
    run = lambda at: attention.cache_read(*cache, at, 64)
    got = torch.func.vmap(run)(slots)
    for i, at in enumerate(slots):
        assert all(torch.equal(g[i], w) for g, w in zip(got, run(at)))
    graph = make_fx(run)(slots[0])
    assert any("cache_read" in str(n.target) for n in graph.graph.nodes)
    assert all(torch.equal(g, w) for g, w in zip(graph(slots[2]), run(slots[2])))


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["token", "head"])
def test_read_of_a_cache_of_16_bits_past_32_bits(layout):
    """A cache of more than 2^32 bytes, read at its ends and where the bytes before pass 2^31 and 2^32."""
    block, heads, dim = 16, 2, 128
    row = heads * dim * 2
    blocks = (1 << 32) // (block * row) + 100
    shape = (blocks, block, heads, dim) if layout == "token" else (blocks, heads, block, dim)
    k, v = (torch.zeros(shape, dtype=HALF, device="cuda") for _ in range(2))
    k, v = (x if layout == "token" else x.transpose(1, 2) for x in (k, v))
    edge = [(1 << 31) // row, (1 << 32) // row]
    slots = torch.tensor([0, edge[0] - 1, edge[0], edge[1] - 1, edge[1], blocks * block - 1, blocks * block, -1], dtype=torch.int32, device="cuda")
    want = torch.randn(2, len(slots), heads, dim, device="cuda").half()
    want[:, -2:] = 0
    for i, s in enumerate(slots.tolist()[:-2]):
        k[s // block, s % block], v[s // block, s % block] = want[0, i], want[1, i]
    for got, w in zip(attention.cache_read(k, v, slots), want):
        assert torch.equal(got, w)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [HALF, BF16])
def test_the_size_of_an_error(dtype):
    """With the group's largest magnitude m in [3.5, 7) 2^e: half a step of the codes is 2^e / 4 up to 2^(e + 1), at most m / 14; above it is
    at most a fifth of the value (from 2.5 to 2, from 5 to 4), and so is what a value beyond 6 2^e loses (7 to 6 is a seventh)."""
    T = 500
    x = torch.randn(T, 2, 128, generator=torch.Generator().manual_seed(3))
    x[:100] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.99] * 16)
    x[100:200] *= 2.0 ** torch.arange(-50, 50)[:, None, None] if dtype == BF16 else 2.0 ** (torch.arange(100)[:, None, None] % 20 - 10)
    x = x.to(dtype)
    cache = empty(T, 1, 2, 128)
    slots = torch.arange(T, dtype=torch.int32, device="cuda")
    attention.cache_write(x.cuda(), x.cuda(), *cache, slots)
    groups = x.double().abs().unflatten(-1, (4, 32))
    bound = torch.maximum(groups.amax(-1, keepdim=True) / 14, groups / 5)
    for back in attention.cache_read(*cache, slots, 128, dtype):
        err = (back.cpu().double() - x.double()).abs().unflatten(-1, (4, 32))
        assert bool((err <= bound).all())
    assert float((err[:100] / groups[:100]).amax()) == 1.0 and bool((err[:100, ..., 6] * 5 == groups[:100, ..., 6]).all())


@pytest.mark.gpu
def test_rows_of_codes_are_those_of_the_heads():
    """Keys of fewer or more groups than the cache's rows, and of as many: which check refuses them."""
    cache = empty(4, 16, 2, 64)
    slots = torch.arange(3, dtype=torch.int32, device="cuda")
    for dim, text in ((32, r"k_codes must be \[blocks, block_size, heads, 16\]"), (96, r"k_codes must be \[blocks, block_size, heads, 48\]"),
                      (128, r"k_codes must be \[blocks, block_size, heads, 64\]")):
        k = torch.zeros(3, 2, dim, device="cuda", dtype=HALF)
        with pytest.raises(RuntimeError, match=text):
            attention.cache_write(k, k, *cache, slots)
        with pytest.raises(RuntimeError, match=text):
            attention.cache_read(*cache, slots, dim)
    k = torch.zeros(3, 2, 40, device="cuda", dtype=HALF)
    attention.cache_write(k, k, *cache, slots)
    assert attention.cache_read(*cache, slots, 40)[0].shape == (3, 2, 40)
