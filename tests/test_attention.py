"""The attention over a paged cache against the same sums in 64 bits."""
import ctypes

import pytest
import torch

from autogptq.tvm_amd import _lib, attention
from tests.attention_util import ROUNDING, Step, assert_attention

HALF, BF16 = torch.float16, torch.bfloat16


def attend(s, **more):
    more = {"max_context": s.most, **more}
    if s.prefix:
        return attention.shared_prefix_attention(s.q, s.k_cache, s.v_cache, s.prefix_blocks, s.prefix, s.tables, s.starts,
                                                 s.contexts, **more)
    return attention.paged_attention(s.q, s.k_cache, s.v_cache, s.tables, s.starts, s.contexts, window=s.window, sinks=s.sinks,
                                     **more)


# (requests, heads, kv_heads, dim, block_size, dtype, layout, window, sinks)
CASES = {
    "one token of one": ([(1, 1)], 1, 1, 64, 16, HALF, "token", 0, 0),
    "single tokens": ([(1, 1), (2, 1), (63, 1), (64, 1), (65, 1), (700, 1)], 8, 2, 128, 16, HALF, "token", 0, 0),
    "single tokens, no shared heads": ([(33, 1), (257, 1), (1030, 1)], 4, 4, 128, 32, BF16, "head", 0, 0),
    "single tokens, sevens": ([(33, 1), (257, 1), (1030, 1)], 14, 2, 128, 7, HALF, "token", 0, 0),
    "sixteen heads share": ([(129, 1), (5, 1)], 16, 1, 128, 16, HALF, "head", 0, 0),
    "twenty-four heads share": ([(129, 1), (500, 1)], 24, 1, 128, 16, HALF, "token", 0, 0),
    "seventy-one heads share": ([(129, 1), (300, 1)], 71, 1, 64, 16, BF16, "token", 0, 0),
    "requests without tokens": ([(5, 0), (9, 1), (0, 0), (40, 2), (7, 0)], 4, 2, 64, 8, HALF, "token", 0, 0),
    "drafts": ([(130, 3), (7, 7), (64, 5), (400, 1)], 8, 4, 128, 16, HALF, "head", 0, 0),
    "drafts of many heads": ([(130, 3), (7, 7), (64, 5), (400, 1)], 16, 2, 128, 16, BF16, "token", 0, 0),
    "window": ([(300, 1), (100, 1), (65, 1), (64, 1)], 8, 2, 128, 16, HALF, "token", 64, 0),
    "window and sinks": ([(300, 1), (100, 1), (65, 1), (66, 1), (3, 1)], 8, 2, 128, 16, HALF, "token", 64, 4),
    "window of one": ([(300, 2), (100, 1), (1, 1)], 4, 2, 64, 16, HALF, "token", 1, 0),
    "more sinks than context": ([(30, 2), (400, 3)], 4, 2, 128, 16, HALF, "token", 9, 50),
    "drafts under a window": ([(300, 5), (70, 9), (20, 20)], 4, 2, 128, 24, HALF, "token", 32, 3),
    "dim 8": ([(300, 1), (70, 40)], 4, 2, 8, 16, HALF, "token", 0, 0),
    "dim 72": ([(300, 1), (70, 3)], 4, 2, 72, 16, HALF, "head", 0, 0),
    "dim 80": ([(300, 1), (90, 1)], 4, 2, 80, 16, BF16, "token", 0, 0),
    "dim 256": ([(300, 1), (90, 2)], 4, 2, 256, 16, HALF, "token", 0, 0),
    "dim 200": ([(300, 1), (90, 2)], 4, 2, 200, 16, BF16, "token", 70, 2),
    "blocks of one": ([(90, 1), (33, 2)], 4, 2, 64, 1, HALF, "token", 0, 0),
    "prompt": ([(200, 200)], 4, 2, 128, 16, HALF, "token", 0, 0),
    "prompts, ragged": ([(1, 1), (129, 129), (64, 64), (333, 200), (17, 3)], 8, 2, 128, 16, BF16, "head", 0, 0),
    "prompts, blocks of 24": ([(500, 250), (33, 33)], 7, 1, 64, 24, HALF, "token", 0, 0),
    "prompts under a window": ([(500, 500), (700, 90), (40, 40)], 4, 2, 128, 16, HALF, "token", 100, 0),
    "prompts under a window with sinks": ([(500, 500), (700, 90), (40, 40)], 4, 1, 128, 16, BF16, "token", 70, 5),
    "prompt under a window with many sinks": ([(600, 600)], 2, 1, 64, 16, HALF, "token", 30, 100),
    "prompt, dim 80": ([(200, 150), (77, 77)], 4, 2, 80, 16, HALF, "token", 0, 0),
    "prompt, dim 256": ([(300, 150), (77, 77)], 4, 2, 256, 16, HALF, "token", 0, 0),
    "prompt, dim 136": ([(300, 150), (77, 77)], 4, 2, 136, 16, BF16, "head", 64, 1),
    "prompts of many heads": ([(70, 70), (9, 9)], 40, 8, 128, 64, HALF, "token", 0, 0),
    "a piece behind a long context": ([(5000, 40)], 4, 1, 128, 16, HALF, "token", 0, 0),
    "prompt, dim 96": ([(300, 150), (77, 77)], 4, 2, 96, 16, HALF, "token", 0, 0),
    "pieces behind long contexts, dim 64": ([(2500, 40), (700, 33)], 4, 1, 64, 16, BF16, "head", 0, 0),
    "pieces behind long contexts, dim 80": ([(2500, 40), (30, 30), (1700, 21)], 7, 1, 80, 24, HALF, "token", 0, 0),
    "pieces behind long contexts, dim 192": ([(2500, 40), (700, 33)], 4, 1, 192, 16, HALF, "token", 0, 0),
    "pieces behind long contexts, dim 256": ([(2500, 40), (700, 33)], 4, 1, 256, 16, BF16, "token", 0, 0),
    "a piece under a long window with sinks": ([(4000, 90)], 4, 1, 128, 16, HALF, "token", 1500, 3),
    "pieces of more requests than a wave": ([(300 + 11 * i, 17 * (i % 3)) for i in range(70)], 4, 1, 64, 16, HALF, "token", 0, 0),
    "one prompt among single tokens": ([(700, 1), (400, 400), (90, 1), (1200, 1)], 4, 1, 128, 16, HALF, "token", 0, 0),
    "long": ([(9000, 1)], 8, 2, 128, 16, HALF, "token", 0, 0),
    "long and short": ([(6000, 1), (3, 1), (900, 1), (1, 1)], 4, 2, 64, 16, BF16, "token", 0, 0),
    "many requests": ([(1 + 7 * i % 50, i % 3) for i in range(200)], 4, 2, 64, 16, HALF, "token", 0, 0),
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(CASES))
def test_attention(name):
    requests, heads, kv_heads, dim, block, dtype, layout, window, sinks = CASES[name]
    s = Step(11, requests, heads, kv_heads, dim, block, dtype, layout, window, sinks)
    got = attend(s)
    assert_attention(got, s, name)
    assert torch.equal(got, attend(s)), "a second call on the same inputs differs"


# (requests, heads, kv_heads, dim, block_size, dtype, prefix)
PREFIXES = {
    "of one token": ([(1, 1), (5, 1)], 4, 2, 64, 16, HALF, 1),
    "small batch": ([(1, 1), (37, 1), (300, 1)], 8, 2, 128, 16, HALF, 1000),
    "own contexts empty": ([(0, 1), (0, 1), (0, 2)], 8, 2, 128, 16, HALF, 130),
    "batch of a few hundred rows": ([(1 + 13 * i % 90, 1) for i in range(70)], 8, 1, 128, 16, BF16, 2100),
    "drafts and requests without tokens": ([(30, 3), (8, 0), (200, 5), (2, 2)], 8, 4, 128, 24, HALF, 777),
    "prompts": ([(150, 150), (64, 30)], 4, 1, 128, 16, HALF, 500),
    "prompts and long own contexts": ([(3000, 60), (64, 30)], 4, 1, 128, 16, HALF, 500),
    "dim 80": ([(20, 1), (90, 2)], 4, 1, 80, 16, BF16, 333),
    "dim 256": ([(20, 1), (90, 2), (400, 40)], 8, 2, 256, 16, HALF, 333),
    "dim 64, sevens": ([(20, 1)] * 9, 7, 1, 64, 7, HALF, 900),
    "long own contexts": ([(3000, 1), (20, 1)], 4, 2, 128, 16, HALF, 200),
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(PREFIXES))
def test_shared_prefix(name):
    requests, heads, kv_heads, dim, block, dtype, prefix = PREFIXES[name]
    s = Step(12, requests, heads, kv_heads, dim, block, dtype, prefix=prefix)
    got = attend(s)
    assert_attention(got, s, name)
    assert torch.equal(got, attend(s))


@pytest.mark.gpu
def test_a_token_that_sees_nothing_gets_zeros():
    # a context that is shorter than the step's tokens: the first of them stand before its beginning
    for counts, heads in (((3, 2), 2), ((200, 1), 4)):
        s = Step(13, [(2, counts[0]), (0, counts[1])], heads, 1, 64, 16)
        got = attend(s)
        assert_attention(got, s, "tokens before the context")
        assert bool((got[:counts[0] - 2] == 0).all()) and bool((got[counts[0]:] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("stale", [-1, 1 << 30, -(1 << 31)])
def test_table_entries_that_nobody_sees_may_hold_anything(stale):
    s = Step(14, [(700, 1), (300, 40), (64, 64)], 4, 2, 64, 16, window=50, sinks=3, stale=stale)
    assert_attention(attend(s), s, f"stale entries {stale}")


@pytest.mark.gpu
def test_values_that_are_large_where_masked():
    # scores of opposite extremes, and the type's largest finite values in slots past the contexts
    s = Step(15, [(77, 1), (130, 130)], 4, 2, 64, 16, q_scale=8.0)
    s.k_cache.nan_to_num_(65504.0)
    s.v_cache.nan_to_num_(65504.0)
    want, size = s.expected()
    got = attend(s)
    # scores reach 64 here: the 32-bit part of the bound grows with them
    assert bool(((got.double() - want).abs() <= 3 * 2.0 ** -11 * size + 2.0 ** -24).all())


@pytest.mark.gpu
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_keys_that_are_not_finite_where_masked(value):
    # the keys of each request's last token, which the tokens before it do not see
    for requests, dim in (([(130, 130), (2000, 50)], 128), ([(70, 4), (5, 2)], 64), ([(200, 60)], 256)):
        s = Step(16, requests, 4, 2, dim, 16)
        want, size = s.expected()
        others = torch.ones(s.tokens, dtype=torch.bool, device=s.q.device)
        for b, (context, _) in enumerate(requests):
            s.k_cache[int(s.tables[b, (context - 1) // 16]), (context - 1) % 16] = value
            others[int(s.starts[b + 1]) - 1] = False
        err = (attend(s).double() - want).abs()
        assert bool((err <= 2.25 * 2.0 ** -11 * size + 2.0 ** -24)[others].all())


@pytest.mark.gpu
@pytest.mark.parametrize("hint", [0, 1, 300, 100000])
def test_max_context_is_a_hint(hint):
    for requests in ([(5000, 1), (40, 1)], [(3000, 60)]):
        s = Step(16, requests, 8, 2, 128, 16)
        assert_attention(attend(s, max_context=hint), s, f"max_context={hint}")


@pytest.mark.gpu
def test_scale():
    s = Step(17, [(200, 1), (50, 50)], 4, 2, 64, 16)
    assert_attention(attend(s, scale=0.03), s, "scale 0.03", scale=0.03)


@pytest.mark.gpu
def test_strided_inputs():
    s = Step(18, [(200, 1), (50, 20)], 8, 2, 64, 16)
    want = attend(s)
    # columns of a fused product, rows apart; a table whose rows are apart; offsets that are not 16-byte aligned
    wide = torch.randn(s.tokens, (8 + 4) * 64, device="cuda").half()
    wide[:, :512] = s.q.reshape(s.tokens, 512)
    tables = torch.zeros(2, s.tables.shape[1] + 5, dtype=torch.int32, device="cuda")
    tables[:, :s.tables.shape[1]] = s.tables
    odd = torch.randn(s.tokens, 8 * 64 + 3, device="cuda").half()
    odd[:, 3:] = s.q.reshape(s.tokens, 512)
    swapped = s.q.transpose(0, 1).contiguous().transpose(0, 1)
    s.tables = tables[:, :s.tables.shape[1]]
    for q in (wide[:, :512].view(s.tokens, 8, 64), odd[:, 3:].view(s.tokens, 8, 64), swapped):
        s.q = q
        assert torch.equal(attend(s), want)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """A cache of more than 2^32 elements whose used blocks lie at its ends."""
    s = Step(19, [(40, 1), (30, 20)], 2, 1, 128, 16)
    want = attend(s)
    blocks = (1 << 32) // (16 * 128) + 4096
    caches = []
    for cache in (s.k_cache, s.v_cache):
        big = torch.empty((blocks, 16, 1, 128), dtype=cache.dtype, device="cuda")
        big[blocks - cache.shape[0]:] = cache
        caches.append(big)
    used = s.tables >= 0
    s.tables = torch.where(used, s.tables + blocks - s.k_cache.shape[0], s.tables)
    s.k_cache, s.v_cache = caches
    assert torch.equal(attend(s), want)
    slots = torch.tensor([blocks * 16 - 1, (blocks - 5) * 16 + 2], dtype=torch.int32, device="cuda")
    k, v = torch.randn(2, 2, 1, 128, device="cuda").half()
    attention.cache_write(k, v, s.k_cache, s.v_cache, slots)
    assert torch.equal(s.k_cache[blocks - 1, 15], k[0]) and torch.equal(s.v_cache[blocks - 5, 2], v[1])


@pytest.mark.gpu
def test_on_another_stream():
    s = Step(20, [(3000, 1), (50, 50)], 4, 2, 128, 16)
    want = attend(s)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = [attend(s) for _ in range(3)]
    side.synchronize()
    assert all(torch.equal(g, want) for g in got)


@pytest.mark.gpu
@pytest.mark.parametrize("prefix, tokens", [(0, 1), (600, 1), (0, 50), (600, 50)])
def test_captured_in_a_graph(prefix, tokens):
    s = Step(21, [(3000, tokens), (50, tokens), (tokens, tokens)], 4, 2, 128, 16, prefix=prefix)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = attend(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = attend(s)
        for _ in range(3):
            got.zero_()
            graph.replay()
            side.synchronize()
            assert torch.equal(got, want)
            assert torch.equal(attend(s), want)     # eager work between the replays
            side.synchronize()


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    s = Step(22, [(40, 1), (30, 20)], 4, 2, 64, 16)
    args = dict(q=s.q, k_cache=s.k_cache, v_cache=s.v_cache, tables=s.tables, starts=s.starts, contexts=s.contexts)
    call = lambda **more: attention.paged_attention(**{**args, **more})
    call()
    for more, text in (
            (dict(q=s.q.bfloat16()), "the cache"), (dict(q=s.q[:, :3]), "multiple"), (dict(q=s.q[..., :32]), r"\[tokens, heads, 64\]"),
            (dict(q=s.q.cpu()), "no CPU fallback"), (dict(v_cache=s.v_cache[:, :8]), "alike"),
            (dict(v_cache=s.v_cache.contiguous().transpose(1, 2).contiguous().transpose(1, 2)), "strides"),
            (dict(k_cache=s.k_cache.float(), v_cache=s.v_cache.float()), "float16 or bfloat16"),
            (dict(tables=s.tables.long()), "int32"), (dict(tables=s.tables[:1]), r"\[2, width\]"),
            (dict(tables=s.tables.t().contiguous().t()), "contiguous"), (dict(starts=s.starts[:2]), "vector of 3"),
            (dict(contexts=s.contexts[::2]), "vector"), (dict(window=-1), "window"), (dict(sinks=-1), "sinks"),
            (dict(max_context=-5), "max_context"), (dict(scale=float("inf")), "scale"),
            (dict(q=s.q.clone().requires_grad_()), "no backward")):
        with pytest.raises(RuntimeError, match=text):
            call(**more)
    for scale in (0.0, -1.0, float("nan")):
        with pytest.raises(ValueError, match="scale"):
            call(scale=scale)
    narrow = s.k_cache[..., :60], s.v_cache[..., :60]
    with pytest.raises(RuntimeError, match="multiple of 8"):
        call(q=s.q[..., :60], k_cache=narrow[0], v_cache=narrow[1])
    with pytest.raises(RuntimeError, match="prefix_blocks has 0"):
        attention.shared_prefix_attention(s.q, s.k_cache, s.v_cache, s.prefix_blocks, 5, s.tables, s.starts, s.contexts)
    assert attention.paged_attention(s.q[:0], s.k_cache, s.v_cache, s.tables[:0], s.starts[:1], s.contexts[:0]).shape == (0, 4, 64)


def test_cpu_tensors_are_refused():
    s = Step(23, [(10, 1)], 2, 1, 64, 16, device="cpu")
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        attend(s)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        attention.cache_write(s.k[0], s.v[0], s.k_cache, s.v_cache, torch.arange(10, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        attention.cache_tables(s.contexts, s.contexts, s.tables, s.contexts, 10, 16)


def plain(**more):
    """A call's description whose pointers are never followed: everything is checked before."""
    a = _lib.Attention()
    a.cache.k = a.cache.v = a.q = a.out = a.tables = a.starts = a.contexts = 0x1000
    values = dict(type=0, blocks=100, block_size=16, heads=8, dim=128, block_stride=16384, slot_stride=1024, head_stride=128)
    for k, v in {**values, **{k: v for k, v in more.items() if k in values or k in ("k", "v")}}.items():
        setattr(a.cache, k, v)
    values = {**dict(tokens=64, requests=64, heads=32, table_width=64, max_context=1000, q_token_stride=4096, q_head_stride=128,
                     table_stride=64, scale=0.1), **more}
    for k, v in values.items():
        if k not in ("type", "blocks", "block_size", "dim", "block_stride", "slot_stride", "head_stride", "k", "v"):
            setattr(a, {"q_heads": "heads"}.get(k, k), v)
    a.cache.heads = 8
    return a


@pytest.mark.parametrize("more, status", [
    (dict(type=2), _lib.ERR_BAD_ARG), (dict(blocks=0), _lib.ERR_BAD_ARG), (dict(block_size=0), _lib.ERR_BAD_ARG),
    (dict(dim=100), _lib.ERR_BAD_ARG), (dict(dim=264), _lib.ERR_UNSUPPORTED), (dict(block_stride=16380), _lib.ERR_BAD_ARG),
    (dict(blocks=1 << 27), _lib.ERR_UNSUPPORTED), (dict(blocks=1 << 22, block_stride=1 << 20), _lib.ERR_UNSUPPORTED),
    (dict(k=0x1008), _lib.ERR_BAD_ARG), (dict(k=None), _lib.ERR_BAD_ARG), (dict(q=0x1004), _lib.ERR_BAD_ARG),
    (dict(out=None), _lib.ERR_BAD_ARG), (dict(starts=None), _lib.ERR_BAD_ARG), (dict(tables=None), _lib.ERR_BAD_ARG),
    (dict(heads=31), _lib.ERR_BAD_ARG), (dict(requests=0), _lib.ERR_BAD_ARG), (dict(tokens=-1), _lib.ERR_BAD_ARG),
    (dict(window=-1), _lib.ERR_BAD_ARG), (dict(scale=0.0), _lib.ERR_BAD_ARG), (dict(scale=float("nan")), _lib.ERR_BAD_ARG),
    (dict(prefix_length=5), _lib.ERR_BAD_ARG), (dict(prefix_length=5, prefix_blocks=0x1000, window=3), _lib.ERR_BAD_ARG),
    (dict(table_stride=63), _lib.ERR_BAD_ARG), (dict(q_token_stride=4100), _lib.ERR_BAD_ARG),
    (dict(tokens=1 << 28), _lib.ERR_UNSUPPORTED)])
def test_the_entry_point_refuses(more, status):
    a = plain(**more)
    assert _lib.lib().gptq_hip_attend(ctypes.byref(a), None, 0, None) == status


def test_workspace():
    lib = _lib.lib()
    a = plain(max_context=30000, table_width=4096, table_stride=4096)
    need = lib.gptq_hip_attention_workspace_bytes(ctypes.byref(a))
    assert need > 65536
    for ws, size in ((None, need), (0x1000, need - 1), (0x1008, need)):
        assert lib.gptq_hip_attend(ctypes.byref(a), ws, size, None) == _lib.ERR_WORKSPACE
    assert lib.gptq_hip_attention_workspace_bytes(None) == 0
    assert lib.gptq_hip_attention_workspace_bytes(ctypes.byref(plain(tokens=0))) == 0
    # a workspace stays within half a GiB of parts whatever the batch
    for tokens, requests, context in ((1, 1, 1 << 20), (256, 256, 1 << 20), (8192, 1, 1 << 17), (4096, 4096, 4096)):
        a = plain(tokens=tokens, requests=requests, max_context=context, table_width=1 << 16, table_stride=1 << 16)
        assert lib.gptq_hip_attention_workspace_bytes(ctypes.byref(a)) <= (1 << 29) + (1 << 20)
    assert lib.gptq_hip_attend(None, None, 0, None) == _lib.ERR_BAD_ARG


@pytest.mark.gpu
def test_through_the_dispatcher():
    """torch.ops.gptq_hip.* and the call in C are the same; tensor subclasses, modes and fake tensors reach the operator."""
    s = Step(24, [(40, 1), (30, 20)], 4, 2, 64, 16)
    want = attend(s)
    args = (s.q, s.k_cache, s.v_cache, s.tables, s.starts, s.contexts, 40, 0, 0, 0.0)
    assert torch.equal(torch.ops.gptq_hip.paged_attention(*args), want)

    class Sub(torch.Tensor):
        pass
    s.q = s.q.as_subclass(Sub)
    assert torch.equal(attend(s).as_subclass(torch.Tensor), want)
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode() as mode:
        fake = [mode.from_tensor(t.as_subclass(torch.Tensor)) if isinstance(t, torch.Tensor) else t for t in args]
        out = torch.ops.gptq_hip.paged_attention(*fake)
        assert out.shape == want.shape and out.dtype == want.dtype
    k, v = torch.randn(2, 3, 2, 64, device="cuda").half()
    before = s.k_cache._version, s.v_cache._version
    attention.cache_write(k, v, s.k_cache, s.v_cache, torch.arange(3, dtype=torch.int32, device="cuda"))
    assert s.k_cache._version > before[0] and s.v_cache._version > before[1]
    with pytest.raises(TypeError):
        attention.paged_attention(s.q, None, s.v_cache, s.tables, s.starts, s.contexts)


def captured(stream, call):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = call()
    return graph, got


def overwrite(n=256 << 20):
    """Fills what the allocator can hand out, on the current stream, with bytes that are no zeros."""
    junk = [torch.full((1 << k,), 0x7f, dtype=torch.uint8, device="cuda") for k in range(9, 28)]
    junk += [torch.full((n // 16,), 0x7f, dtype=torch.uint8, device="cuda") for _ in range(16)]
    return junk


@pytest.mark.gpu
@pytest.mark.parametrize("heads, kv_heads", [(4, 2), (32, 8)])
def test_a_captured_call_does_not_depend_on_later_calls(heads, kv_heads):
    """Eager calls that need more workspace than a captured one come after it on its stream; what they leave behind is
    overwritten."""
    small = Step(31, [(2000, 1), (700, 1)], heads, kv_heads, 128, 16)
    large = Step(32, [(6000, 500)], heads, kv_heads, 128, 16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want, other = attend(small), attend(large)
        del other
        torch.cuda.empty_cache()
    # a stream whose workspace has the small call's size
    stream = torch.cuda.Stream()
    stream.wait_stream(side)
    with torch.cuda.stream(stream):
        attend(small)
        graph, got = captured(stream, lambda: attend(small))
        for _ in range(3):
            attend(large)
            junk = overwrite()
            got.zero_()
            graph.replay()
            stream.synchronize()
            assert torch.equal(got, want)
            assert all(bool((j == 0x7f).all()) for j in junk), "a replay wrote into another tensor"
            del junk


@pytest.mark.gpu
def test_captures_replay_in_any_order():
    """Two captures on one stream that was not warmed up: the second is replayed first, and each with the other's parts in
    between."""
    steps = [Step(33, [(2000, 1), (700, 1)], 8, 2, 128, 16), Step(34, [(3000, 1), (90, 1), (1500, 2)], 8, 2, 128, 16),
             Step(35, [(3000, 60)], 8, 2, 128, 16, prefix=0)]
    want = [attend(s) for s in steps]
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    junk = overwrite()      # (what new pools get is not zero by chance)
    del junk
    torch.cuda.empty_cache()
    made = [captured(stream, lambda s=s: attend(s)) for s in steps]
    for order in ((1, 0, 2), (2, 1, 0), (0, 0, 1), (1, 2, 2)):
        for i in order:
            made[i][1].zero_()
            made[i][0].replay()
        torch.cuda.synchronize()
        for i in set(order):
            assert torch.equal(made[i][1], want[i]), (order, i)


@pytest.mark.gpu
def test_two_captures_replay_on_two_streams_at_once():
    steps = [Step(36, [(4000, 1), (700, 1)], 8, 2, 128, 16), Step(37, [(3000, 1), (90, 1), (2500, 1)], 8, 2, 128, 16)]
    want = [attend(s) for s in steps]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for s in steps:
            attend(s)
    made = [captured(stream, lambda s=s: attend(s)) for s in steps]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in made]
    for _ in range(20):
        for (graph, got), s in zip(made, streams):
            with torch.cuda.stream(s):
                got.zero_()
                graph.replay()
        torch.cuda.synchronize()
        for (_, got), w in zip(made, want):
            assert torch.equal(got, w)


@pytest.mark.gpu
def test_a_capture_that_grows_its_workspace():
    steps = [Step(38, [(2000, 1)], 4, 2, 128, 16), Step(39, [(6000, 500)], 32, 8, 128, 16), Step(40, [(2500, 1), (40, 1)], 32, 8, 128, 16)]
    want = [attend(s) for s in steps]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph, got = captured(stream, lambda: [attend(s) for s in steps])
    for _ in range(3):
        for g in got:
            g.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for g, w in zip(got, want))


def one_high_key(s, gap, at):
    """Key `at` of every request (of the prefix and its context together) lies `gap` octaves above all others and has no value: the
    output is what the others' small shares make of it."""
    gen = torch.Generator().manual_seed(41)
    noise = lambda *shape: (torch.randn(*shape, generator=gen) * 0.25).to(s.dtype).to(s.q.device)
    s.q = noise(*s.q.shape)
    s.q[..., 0] = 4.0
    front = noise(s.prefix, s.kv_heads, s.dim)
    for b, (c, _) in enumerate(s.requests):
        s.k[b] = torch.cat([front, noise(c, s.kv_heads, s.dim)])
        s.k[b][..., 0] = 0.0
        s.k[b][at] = 0.0
        s.k[b][at, :, 0] = gap * 0.6931 * s.dim ** 0.5 / 4
        s.v[b][at] = 0.0
        p, blocks = s.prefix, -(-c // s.block_size)
        s._fill(s.prefix_blocks, s.k[b][:p], s.v[b][:p], 0)
        s._fill(s.tables[b, :blocks], s.k[b][p:], s.v[b][p:], 0)
    return s


@pytest.mark.gpu
@pytest.mark.parametrize("gap", [16.0, 22.3, 24.6])
@pytest.mark.parametrize("requests, dim, dtype, prefix, at", [
    ([(30000, 1)], 128, HALF, 0, 0), ([(9000, 1), (300, 1)], 64, HALF, 0, 3), ([(3000, 1), (500, 2)], 256, HALF, 0, 299),
    ([(9000, 40)], 128, HALF, 0, 0), ([(2000, 90), (150, 60)], 64, HALF, 0, 5), ([(3000, 50)], 256, HALF, 0, 1000),
    ([(400, 300)], 80, HALF, 0, 0), ([(20, 1), (900, 1)] * 3, 128, HALF, 9000, 0), ([(20, 1), (900, 1)], 128, HALF, 300, 250),
    ([(300, 40)] * 3, 128, HALF, 3000, 2), ([(9000, 1)], 128, BF16, 0, 0), ([(9000, 40)], 128, BF16, 0, 0)])
def test_shares_far_below_the_largest(requests, dim, dtype, prefix, at, gap):
    """(One key holds nearly all of every row: what remains has shares of 2^-16 to 2^-25 of it, and makes the output.)"""
    s = one_high_key(Step(40, requests, 4, 2, dim, 16, dtype, prefix=prefix), gap, at)
    assert_attention(attend(s), s, f"{gap} octaves")


@pytest.mark.gpu
@pytest.mark.parametrize("requests, heads, kv_heads, dim, prefix", [
    ([(40, 1), (700, 1)], 8, 2, 128, 0), ([(5, 0), (0, 0)], 4, 2, 64, 0), ([(3, 1)], 7, 1, 72, 0), ([(40, 3), (7, 2)], 16, 2, 128, 0),
    ([(300, 300)], 4, 2, 128, 0), ([(3000, 60), (64, 64)], 4, 1, 64, 0), ([(300, 150)], 4, 2, 256, 0),
    ([(40, 1), (30, 1)], 8, 2, 128, 100), ([(40, 1), (30, 1)], 8, 2, 128, 9000), ([(300, 90)], 8, 1, 80, 3000)])
@pytest.mark.parametrize("ahead, behind", [(0, 1), (0, 300), (3, 5)])
def test_tokens_of_no_request_get_zeros(requests, heads, kv_heads, dim, prefix, ahead, behind):
    s = Step(42, requests, heads, kv_heads, dim, 16, prefix=prefix)
    want, size = s.expected()
    n = s.tokens
    s.q = torch.cat([torch.full((ahead, heads, dim), float("nan"), device="cuda").half(), s.q,
                     torch.full((behind, heads, dim), float("nan"), device="cuda").half()])
    s.starts += ahead
    torch.full(s.q.shape, float("nan"), dtype=s.dtype, device="cuda")      # what the result's memory holds
    got = attend(s)
    assert bool((got[:ahead] == 0).all()) and bool((got[ahead + n:] == 0).all())
    assert bool(((got[ahead:ahead + n].double() - want).abs() <= 2.25 * ROUNDING[s.dtype] * size + 2.0 ** -24).all())


@pytest.mark.gpu
@pytest.mark.parametrize("requests", [[(300, 1), (70, 1)], [(130, 3), (40, 2)], [(300, 150)]])
@pytest.mark.parametrize("dim", [8, 40, 64, 72, 96, 128, 200, 256])
def test_a_key_that_is_minus_infinity_has_no_share(dim, requests):
    """(In its last dimension, where the products of widths that are no power of two end.)"""
    s = Step(43, requests, 4, 2, dim, 16)
    s.q[..., -1] = s.q[..., -1].abs() + 0.125
    for b in range(len(requests)):
        for j in (5, 33):
            s.k[b][j, :, -1] = -float("inf")
            s.k_cache[int(s.tables[b, j // 16]), j % 16, :, -1] = -float("inf")
    assert_attention(attend(s), s, "a key of minus infinity")


def test_assembly_declares_what_it_writes():
    """Requests into LDS write m0: the compiler must know."""
    import os
    import re
    csrc = os.path.dirname(_lib.LIB_PATH)
    seen = 0
    for name in os.listdir(csrc):
        if name.startswith("gptq_attention"):
            with open(os.path.join(csrc, name), encoding="utf-8") as f:
                for statement in re.findall(r"asm volatile\(.*?\);", f.read(), re.S):
                    if re.search(r"\bm0, ", statement):
                        seen += 1
                        assert '"m0"' in statement, (name, statement)
    assert seen == 1


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["k_cache", "v_cache"])
def test_caches_that_require_grad_are_refused(which):
    s = Step(44, [(40, 1), (30, 20)], 4, 2, 64, 16, prefix=20)
    setattr(s, which, getattr(s, which).clone().requires_grad_())
    k, v = torch.randn(2, 3, 2, 64, device="cuda").half()
    slots = torch.arange(3, dtype=torch.int32, device="cuda")
    calls = (lambda: attend(s), lambda: attention.cache_write(k, v, s.k_cache, s.v_cache, slots),
             lambda: attention.paged_attention(s.q, s.k_cache, s.v_cache, s.tables, s.starts, s.contexts),
             lambda: torch.ops.gptq_hip.cache_write(k, v, s.k_cache, s.v_cache, slots))
    for call in calls:
        with pytest.raises(RuntimeError, match=f"{which} requires grad"):
            call()
        with torch.no_grad():
            call()


def test_meta_tensors_have_a_shape():
    s = Step(45, [(40, 1), (30, 20)], 4, 2, 64, 16, device="cpu")
    meta = lambda t: t.to("meta")
    out = attention.paged_attention(*map(meta, (s.q, s.k_cache, s.v_cache, s.tables, s.starts, s.contexts)))
    assert out.device.type == "meta" and out.shape == s.q.shape and out.dtype == s.q.dtype
    made = attention.cache_tables(meta(s.contexts), meta(s.contexts), meta(s.tables), meta(s.contexts), 21, 16)
    assert [len(x) for x in made] == [3, 2, 21, 21, 1]
    k = torch.zeros(3, 2, 64, dtype=HALF, device="meta")
    assert attention.cache_write(k, k, meta(s.k_cache), meta(s.v_cache), meta(torch.arange(3, dtype=torch.int32))) is None


@pytest.mark.gpu
def test_function_modes_and_transforms_see_the_operators():
    from torch.overrides import TorchFunctionMode

    s = Step(46, [(40, 1), (30, 20)], 4, 2, 64, 16)
    rest = (s.k_cache, s.v_cache, s.tables, s.starts, s.contexts)
    want = attend(s)

    class Mode(TorchFunctionMode):
        seen = []

        def __torch_function__(self, func, types, args=(), kwargs=None):
            self.seen.append(str(func))
            return func(*args, **(kwargs or {}))
    with Mode():
        got = attend(s)
        attention.cache_write(s.k_cache[0, :3], s.v_cache[0, :3], s.k_cache, s.v_cache, torch.full((3,), -1, dtype=torch.int32, device="cuda"))
        attention.cache_tables(s.contexts, s.contexts, s.tables.clone(), s.contexts, 70, 16)
    assert torch.equal(got, want)
    for name in ("paged_attention", "cache_write", "cache_tables"):
        assert any(name in f for f in Mode.seen), (name, Mode.seen)
    qs = torch.stack([s.q, s.q * 0.5, s.q.flip(0)])
    got = torch.func.vmap(lambda q: attention.paged_attention(q, *rest))(qs)
    assert got.shape == qs.shape
    for g, q in zip(got, qs):
        assert torch.equal(g, attention.paged_attention(q, *rest))
