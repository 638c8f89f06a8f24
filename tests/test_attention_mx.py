"""The attention over a cache in MXFP4 against the same sums in 64 bits over what the codes stand for."""
import ctypes

import pytest
import torch

from autogptq.tvm_amd import _lib, attention
from autogptq.tvm_amd.attention import Mxfp4
from tests.attention_util import ROUNDING, Step, assert_attention
from tests.mxfp4_util import MxStep, decode, encode
from tests.test_attention import CASES, PREFIXES, attend, captured, overwrite

HALF, BF16 = torch.float16, torch.bfloat16

MORE = {     # widths whose last group is not whole, or that leave groups of the kernels' rows out; heads in both layouts
    "dim 32": ([(300, 1), (70, 40)], 4, 2, 32, 16, HALF, "head", 0, 0),
    "dim 40": ([(300, 1), (5, 2)], 4, 2, 40, 16, BF16, "head", 0, 0),
    "dim 96": ([(300, 1), (90, 2)], 4, 2, 96, 16, HALF, "head", 0, 0),
    "dim 104": ([(300, 2), (90, 1)], 4, 2, 104, 16, BF16, "token", 0, 0),
    "dim 136": ([(300, 1), (90, 2)], 4, 2, 136, 16, HALF, "head", 0, 0),
    "dim 160": ([(300, 1), (90, 2)], 4, 2, 160, 16, BF16, "head", 64, 3),
    "dim 232": ([(300, 1), (90, 2)], 4, 2, 232, 16, HALF, "token", 0, 0),
    "prompt, dim 40": ([(200, 150), (77, 77)], 4, 2, 40, 16, HALF, "head", 0, 0),
    "prompt, dim 160": ([(200, 150), (77, 77)], 4, 2, 160, 16, BF16, "head", 0, 0),
    "prompt, dim 200": ([(200, 150), (77, 77)], 4, 2, 200, 16, HALF, "token", 30, 2),
    "prompt, dim 224": ([(200, 150), (77, 77)], 4, 2, 224, 16, HALF, "head", 0, 0),
    "single tokens, dim 256": ([(1000, 1), (31, 1), (260, 1)], 8, 2, 256, 16, HALF, "head", 0, 0),
    "single tokens, lengths around a wave's blocks": ([(n, 1) for n in (31, 32, 33, 127, 128, 129, 255, 256, 257, 383, 385, 511, 513)],
                                                      4, 2, 128, 16, HALF, "head", 0, 0),
    "one long context alone": ([(20000, 1)], 4, 1, 128, 64, HALF, "head", 0, 0),
    "two operands": ([(900, 1), (1300, 1), (40, 1)], 24, 1, 128, 16, BF16, "head", 0, 0),
    "ragged pieces behind long contexts": ([(7000, 60), (300, 40), (2500, 130), (6500, 1), (0, 0)], 4, 1, 128, 16, HALF, "head", 0, 0),
    "ragged pieces behind long contexts, dim 64": ([(9000, 33), (9000, 32), (128, 128), (5000, 70)], 8, 2, 64, 64, BF16, "head", 0, 0),
    "ragged pieces behind long contexts, dim 256": ([(6200, 50), (640, 40), (6300, 30)], 4, 1, 256, 16, HALF, "head", 0, 0),
    "ragged pieces under a long window": ([(9000, 60), (300, 40), (12000, 130)], 4, 1, 128, 24, HALF, "head", 7000, 5),
    "more tiles than workgroups behind long contexts": ([(6400 - 700 * (i % 9), 64) for i in range(40)], 32, 4, 64, 64, HALF, "head", 0, 0),
    "single tokens beside a piece": ([(1 + 397 * i % 6000, 1) for i in range(40)] + [(3000, 300), (50, 50), (0, 0), (2000, 4), (2000, 5)], 8, 2, 64, 16, HALF, "head", 0, 0),
    "single tokens beside a piece, dim 128": ([(7000, 70)] + [(8100 - 97 * i, 1) for i in range(20)] + [(6300, 3), (0, 0)], 16, 4, 128, 64, BF16, "head", 0, 0),
    "single tokens beside a piece, window": ([(9000, 1)] * 6 + [(9000, 200), (200, 200)] + [(7777, 1)] * 3, 24, 8, 80, 24, HALF, "head", 6500, 3),
    "single tokens beside a piece, dim 256": ([(6200 - 211 * i, 1) for i in range(20)] + [(6400, 2), (6300, 60), (6500, 1)], 8, 4, 256, 16, HALF, "head", 0, 0),
    "single tokens beside pieces, many requests": ([(2500 - 7 * i, 1) for i in range(80)] + [(2000, 400), (64, 64)] + [(1, 1)] * 10 + [(900, 700)], 16, 4, 64, 16, HALF, "head", 0, 0),
    "heads that fit no few rows": ([(8200, 1)] * 12 + [(3000, 40)], 35, 1, 64, 16, HALF, "head", 0, 0),
    "two operands, dim 64": ([(900, 7), (1300, 5), (40, 7)], 4, 1, 64, 16, HALF, "head", 0, 0),
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(CASES) + ["more: " + n for n in MORE])
def test_attention(name):
    requests, heads, kv_heads, dim, block, dtype, layout, window, sinks = CASES[name] if name in CASES else MORE[name[6:]]
    s = MxStep(11, requests, heads, kv_heads, dim, block, dtype, layout, window, sinks)
    got = attend(s)
    assert_attention(got, s, name)
    assert torch.equal(got, attend(s)), "a second call on the same inputs differs"


LONG_PREFIXES = {
    "ragged pieces behind long contexts": ([(6500, 40), (300, 40), (2500, 130)], 4, 1, 128, 16, HALF, 700),
    "single tokens beside a piece": ([(3000 + 61 * i, 1) for i in range(30)] + [(2000, 200), (300, 300)], 16, 4, 128, 16, BF16, 5000),
    "tiles in two a CU": ([(1 + i % 7, 1) for i in range(64)], 64, 8, 64, 64, HALF, 16500),
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(PREFIXES) + ["long: " + n for n in LONG_PREFIXES])
def test_shared_prefix(name):
    requests, heads, kv_heads, dim, block, dtype, prefix = PREFIXES[name] if name in PREFIXES else LONG_PREFIXES[name[6:]]
    s = MxStep(12, requests, heads, kv_heads, dim, block, dtype, prefix=prefix)
    got = attend(s)
    assert_attention(got, s, name)
    assert torch.equal(got, attend(s))


@pytest.mark.gpu
def test_a_token_that_sees_nothing_gets_zeros():
    for counts, heads in (((3, 2), 2), ((200, 1), 4)):
        s = MxStep(13, [(2, counts[0]), (0, counts[1])], heads, 1, 64, 16)
        got = attend(s)
        assert_attention(got, s, "tokens before the context")
        assert bool((got[:counts[0] - 2] == 0).all()) and bool((got[counts[0]:] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("stale", [-1, 1 << 30, -(1 << 31)])
def test_table_entries_that_nobody_sees_may_hold_anything(stale):
    s = MxStep(14, [(700, 1), (300, 40), (64, 64)], 4, 2, 64, 16, window=50, sinks=3, stale=stale)
    assert_attention(attend(s), s, f"stale entries {stale}")


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 80, 128, 200, 256])
@pytest.mark.parametrize("requests", [[(130, 130), (2000, 50)], [(70, 4), (5, 2)]])
def test_keys_that_are_nan_where_masked(dim, requests):
    """(The keys of each request's last token, which the tokens before it do not see.)"""
    s = MxStep(16, requests, 4, 2, dim, 16)
    want, size = s.expected()
    others = torch.ones(s.tokens, dtype=torch.bool, device=s.q.device)
    for b, (context, _) in enumerate(requests):
        s.k_cache.scales[int(s.tables[b, (context - 1) // 16]), (context - 1) % 16] = 255
        others[int(s.starts[b + 1]) - 1] = False
    got = attend(s)
    assert bool(((got.double() - want).abs() <= 2.25 * 2.0 ** -11 * size + 2.0 ** -24)[others].all())
    assert bool(got[~others].isnan().all())


@pytest.mark.gpu
@pytest.mark.parametrize("requests, dim", [([(300, 1), (70, 2)], 80), ([(300, 1)], 40), ([(300, 1)], 200), ([(200, 150)], 80), ([(200, 150)], 40),
                                           ([(200, 150)], 200)])
def test_what_lies_behind_a_row_does_not_count(requests, dim):
    """Codes behind dim and scales behind the last group, and codes behind it within the last."""
    s = MxStep(47, requests, 4, 2, dim, 16)
    want = attend(s)
    groups = -(-dim // 32)
    for c in (s.k_cache, s.v_cache):
        c.scales[..., groups:] = torch.randint(0, 256, c.scales[..., groups:].shape, device="cuda").to(torch.uint8)
        c.codes[..., dim // 2:] = torch.randint(0, 256, c.codes[..., dim // 2:].shape, device="cuda").to(torch.uint8)
    assert torch.equal(attend(s), want)


@pytest.mark.gpu
@pytest.mark.parametrize("hint", [0, 1, 300, 100000])
def test_max_context_is_a_hint(hint):
    for requests in ([(5000, 1), (40, 1)], [(3000, 60)]):
        s = MxStep(16, requests, 8, 2, 128, 16)
        assert_attention(attend(s, max_context=hint), s, f"max_context={hint}")


@pytest.mark.gpu
def test_scale():
    s = MxStep(17, [(200, 1), (50, 50)], 4, 2, 64, 16)
    assert_attention(attend(s, scale=0.03), s, "scale 0.03", scale=0.03)


@pytest.mark.gpu
def test_strided_inputs():
    s = MxStep(18, [(200, 1), (50, 20)], 8, 2, 64, 16)
    want = attend(s)
    wide = torch.randn(s.tokens, (8 + 4) * 64, device="cuda").half()
    wide[:, :512] = s.q.reshape(s.tokens, 512)
    tables = torch.zeros(2, s.tables.shape[1] + 5, dtype=torch.int32, device="cuda")
    tables[:, :s.tables.shape[1]] = s.tables
    odd = torch.randn(s.tokens, 8 * 64 + 3, device="cuda").half()
    odd[:, 3:] = s.q.reshape(s.tokens, 512)
    s.tables = tables[:, :s.tables.shape[1]]
    # codes and scales of a row in one record of 48 bytes, heads among others
    blocks = s.k_cache.codes.shape[0]
    records = [torch.full((blocks, 16, 5, 48), 0xFF, dtype=torch.uint8, device="cuda") for _ in range(2)]
    for r, c in zip(records, (s.k_cache, s.v_cache)):
        r[:, :, 1:3, :32], r[:, :, 1:3, 32:34] = c.codes, c.scales
    caches = [[Mxfp4(r[:, :, 1:3, :32], r[:, :, 1:3, 32:34]) for r in records], [s.k_cache, s.v_cache]]
    for s.k_cache, s.v_cache in caches:
        for q in (wide[:, :512].view(s.tokens, 8, 64), odd[:, 3:].view(s.tokens, 8, 64), s.q.transpose(0, 1).contiguous().transpose(0, 1)):
            s.q = q
            assert torch.equal(attend(s), want)


@pytest.mark.gpu
@pytest.mark.parametrize("requests", [[(40, 1), (30, 2)], [(40, 1), (300, 200)]])
def test_offsets_past_32_bits(requests):
    """A cache of more than 2^32 bytes whose used blocks lie at its ends."""
    s = MxStep(19, requests, 2, 1, 128, 16)
    want = attend(s)
    used = s.k_cache.codes.shape[0]
    blocks = (1 << 32) // (16 * 64) + 4096
    made = attention.mxfp4_cache(blocks, 16, 1, 128)
    for big, c in zip(made, (s.k_cache, s.v_cache)):
        big.codes[blocks - used:], big.scales[blocks - used:] = c.codes, c.scales
    s.tables = torch.where(s.tables >= 0, s.tables + blocks - used, s.tables)
    s.k_cache, s.v_cache = made
    assert torch.equal(attend(s), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, low, high", [(HALF, -20, 5), (BF16, -60, 10)])
@pytest.mark.parametrize("requests", [[(500, 1), (20, 1)], [(500, 120)]])
def test_groups_of_very_different_sizes(requests, dtype, low, high):
    """Every group's exponent is its own, subnormal values of fp16 among them.  (Queries small enough for scores below 16.)"""
    s = MxStep(48, requests, 4, 2, 128, 16, dtype)
    gen = torch.Generator().manual_seed(9)
    s.q *= 2.0 ** -high / 8
    for which in ("k", "v"):
        cache = getattr(s, which + "_cache")
        e = torch.randint(low, high + 1, cache.scales.shape, generator=gen).cuda()
        cache.scales.copy_(torch.where(cache.scales == 255, 255, e + 125))
        rows = []
        for b, (c, _) in enumerate(requests):
            at = torch.arange(c, device="cuda")
            block = s.tables[b].long()[at // 16]
            rows.append(decode(cache.codes[block, at % 16], cache.scales[block, at % 16], 128))
        setattr(s, which, rows)
    assert_attention(attend(s), s, "sizes")


@pytest.mark.gpu
@pytest.mark.parametrize("prefix, tokens", [(0, 1), (600, 1), (9000, 2), (0, 50), (600, 50)])
def test_captured_in_a_graph(prefix, tokens):
    s = MxStep(21, [(3000, tokens), (50, tokens), (tokens, tokens)], 4, 2, 128, 16, prefix=prefix)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = attend(s)
        graph, got = captured(side, lambda: attend(s))
        for _ in range(3):
            got.zero_()
            graph.replay()
            side.synchronize()
            assert torch.equal(got, want)
            assert torch.equal(attend(s), want)     # eager work between the replays
            side.synchronize()


@pytest.mark.gpu
def test_captures_beside_larger_calls_and_plain_caches():
    """Eager calls that need more workspace, on both kinds of caches, between the replays of two captures."""
    steps = [MxStep(33, [(2000, 1), (700, 1)], 8, 2, 128, 16), MxStep(34, [(3000, 60)], 8, 2, 128, 16)]
    large = [MxStep(35, [(6000, 500)], 32, 8, 128, 16), Step(36, [(6000, 1), (4000, 1)], 32, 8, 128, 16)]
    want, other = [attend(s) for s in steps], [attend(s) for s in large]
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    made = [captured(stream, lambda s=s: attend(s)) for s in steps]
    for order in ((1, 0), (0, 0), (0, 1)):
        with torch.cuda.stream(stream):
            assert all(torch.equal(attend(s), w) for s, w in zip(large, other))
            junk = overwrite()
            for i in order:
                made[i][1].zero_()
                made[i][0].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(made[i][1], want[i]) for i in set(order))
        assert all(bool((j == 0x7f).all()) for j in junk), "a replay wrote into another tensor"
        del junk


@pytest.mark.gpu
@pytest.mark.parametrize("requests, heads, kv_heads, dim, prefix", [
    ([(40, 1), (700, 1)], 8, 2, 128, 0), ([(5, 0), (0, 0)], 4, 2, 64, 0), ([(300, 300)], 4, 2, 128, 0), ([(3000, 60), (64, 64)], 4, 1, 64, 0),
    ([(40, 1), (30, 1)], 8, 2, 128, 9000), ([(300, 90)], 8, 1, 80, 3000)])
@pytest.mark.parametrize("ahead, behind", [(0, 300), (3, 5)])
def test_tokens_of_no_request_get_zeros(requests, heads, kv_heads, dim, prefix, ahead, behind):
    s = MxStep(42, requests, heads, kv_heads, dim, 16, prefix=prefix)
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
def test_write_then_attend():
    """A step as a program makes it: tables, write, attention; single tokens behind a prompt."""
    gen = torch.Generator().manual_seed(8)
    k_cache, v_cache = attention.mxfp4_cache(40, 16, 2, 80)
    tables = torch.full((2, 20), -1, dtype=torch.int32, device="cuda")
    free = torch.randperm(40, generator=gen).to(torch.int32).cuda()
    lengths = torch.zeros(2, dtype=torch.int32, device="cuda")
    seen = [[], []]
    for counts in ((100, 33), (1, 1), (1, 0), (3, 20)):
        n = sum(counts)
        made = attention.cache_tables(lengths, torch.tensor(counts, dtype=torch.int32, device="cuda"), tables, free, n, 16)
        free, lengths = free[int(made.taken):], made.contexts
        q, k, v = (torch.randn(n, h, 80, generator=gen).to(BF16).cuda() for h in (6, 2, 2))
        attention.cache_write(k, v, k_cache, v_cache, made.slots)
        got = attention.paged_attention(q, k_cache, v_cache, tables, made.starts, made.contexts)
        for b in (0, 1):
            seen[b].append((k, v, slice(int(made.starts[b]), int(made.starts[b + 1]))))
        s = Step.__new__(Step)
        s.requests, s.window, s.sinks, s.prefix, s.dim, s.heads, s.kv_heads, s.dtype = list(zip(lengths.tolist(), counts)), 0, 0, 0, 80, 6, 2, BF16
        s.q, s.tokens = q, n
        s.k, s.v = ([torch.cat([decode(*encode(x[which][x[2]]), 80) for x in seen[b]]) for b in (0, 1)] for which in (0, 1))
        assert_attention(got, s, f"counts {counts}")


def test_the_entry_point_refuses():
    lib, p = _lib.lib(), 0x1000

    def call(workspace=None, size=0, **more):
        c = dict(k=p, v=p, k_scales=p, v_scales=p, type=0, blocks=100, block_size=16, heads=8, dim=128, block_stride=8192, slot_stride=512,
                 head_stride=64, scale_block_stride=512, scale_slot_stride=32, scale_head_stride=4)
        cache = _lib.CacheMx(**{**c, **{k: v for k, v in more.items() if k in c}})
        a = _lib.Attention()
        a.q = a.out = a.tables = a.starts = a.contexts = p
        values = dict(tokens=64, requests=64, heads=32, table_width=64, max_context=1000, q_token_stride=4096, q_head_stride=128, table_stride=64,
                      scale=0.1)
        for k, v in {**values, **{k: v for k, v in more.items() if k not in c}}.items():
            setattr(a, {"q_heads": "heads"}.get(k, k), v)
        return (lib.gptq_hip_attend_mx(ctypes.byref(cache), ctypes.byref(a), workspace, size, None),
                lib.gptq_hip_attention_mx_workspace_bytes(ctypes.byref(cache), ctypes.byref(a)))
    for more, status in ((dict(type=2), _lib.ERR_BAD_ARG), (dict(dim=100), _lib.ERR_BAD_ARG), (dict(dim=264), _lib.ERR_UNSUPPORTED),
                         (dict(k_scales=None), _lib.ERR_BAD_ARG), (dict(v_scales=p + 2), _lib.ERR_BAD_ARG), (dict(k=p + 8), _lib.ERR_BAD_ARG),
                         (dict(slot_stride=520), _lib.ERR_BAD_ARG), (dict(scale_head_stride=2), _lib.ERR_BAD_ARG),
                         (dict(blocks=1 << 27), _lib.ERR_UNSUPPORTED), (dict(q=p + 4), _lib.ERR_BAD_ARG), (dict(out=None), _lib.ERR_BAD_ARG),
                         (dict(starts=None), _lib.ERR_BAD_ARG), (dict(q_heads=31), _lib.ERR_BAD_ARG), (dict(requests=0), _lib.ERR_BAD_ARG),
                         (dict(tokens=-1), _lib.ERR_BAD_ARG), (dict(scale=float("nan")), _lib.ERR_BAD_ARG), (dict(prefix_length=5), _lib.ERR_BAD_ARG),
                         (dict(prefix_length=5, prefix_blocks=p, window=3), _lib.ERR_BAD_ARG), (dict(table_stride=63), _lib.ERR_BAD_ARG),
                         (dict(tokens=1 << 28), _lib.ERR_UNSUPPORTED)):
        assert call(**more) == (status, 0), more
    assert call()[0] == _lib.ERR_WORKSPACE and call()[1] > 65536
    need = call()[1]
    for workspace, size in ((None, need), (p, need - 1), (p + 8, need)):
        assert call(workspace, size)[0] == _lib.ERR_WORKSPACE
    assert call(tokens=0) == (_lib.OK, 0)
    assert lib.gptq_hip_attend_mx(None, None, None, 0, None) == _lib.ERR_BAD_ARG
    assert lib.gptq_hip_attention_mx_workspace_bytes(None, None) == 0


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    s = MxStep(22, [(40, 1), (30, 20)], 4, 2, 64, 16)
    args = dict(q=s.q, k_cache=s.k_cache, v_cache=s.v_cache, tables=s.tables, starts=s.starts, contexts=s.contexts)
    call = lambda **more: attention.paged_attention(**{**args, **more})
    call()
    swap = lambda c, **more: c._replace(**more)
    for more, text in (
            (dict(q=s.q.float()), "float16 or bfloat16"), (dict(q=s.q[:, :3]), "multiple"), (dict(q=s.q[..., :32]), "k_codes must be"),
            (dict(q=s.q.cpu()), "no CPU fallback"), (dict(v_cache=swap(s.v_cache, codes=s.v_cache.codes[:, :8])), "same"),
            (dict(k_cache=swap(s.k_cache, scales=s.k_cache.scales.int())), "uint8"),
            (dict(tables=s.tables.long()), "int32"), (dict(starts=s.starts[:2]), "vector of 3"), (dict(window=-1), "window"),
            (dict(max_context=-5), "max_context"), (dict(scale=float("inf")), "scale"), (dict(q=s.q.clone().requires_grad_()), "no backward")):
        with pytest.raises(RuntimeError, match=text):
            call(**more)
    with pytest.raises(TypeError, match="both be"):
        call(v_cache=s.v_cache.codes)
    with pytest.raises(RuntimeError, match="prefix_blocks has 0"):
        attention.shared_prefix_attention(s.q, s.k_cache, s.v_cache, s.prefix_blocks, 5, s.tables, s.starts, s.contexts)
    assert attention.paged_attention(s.q[:0], s.k_cache, s.v_cache, s.tables[:0], s.starts[:1], s.contexts[:0]).shape == (0, 4, 64)


def test_cpu_tensors_are_refused_and_meta_tensors_have_a_shape():
    s = MxStep(23, [(10, 1)], 2, 1, 64, 16, device="cpu", prefix=20)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        attend(s)
    s.q, s.tables, s.starts, s.contexts, s.prefix_blocks = (t.to("meta") for t in (s.q, s.tables, s.starts, s.contexts, s.prefix_blocks))
    s.k_cache, s.v_cache = (Mxfp4(*(t.to("meta") for t in c)) for c in (s.k_cache, s.v_cache))
    for s.prefix in (20, 0):
        out = attend(s)
        assert out.device.type == "meta" and out.shape == s.q.shape and out.dtype == s.q.dtype


@pytest.mark.gpu
def test_through_the_dispatcher():
    from torch.overrides import TorchFunctionMode

    for prefix in (0, 30):
        s = MxStep(24, [(40, 1), (30, 20)], 4, 2, 64, 16, prefix=prefix)
        want = attend(s)
        rest = (*s.k_cache, *s.v_cache, *([s.prefix_blocks, prefix] if prefix else []), s.tables, s.starts, s.contexts, 40)
        op = torch.ops.gptq_hip.shared_prefix_attention_mx if prefix else torch.ops.gptq_hip.paged_attention_mx
        assert torch.equal(op(s.q, *rest, 0.0) if prefix else op(s.q, *rest, 0, 0, 0.0), want)

        class Mode(TorchFunctionMode):
            seen = []

            def __torch_function__(self, func, types, args=(), kwargs=None):
                self.seen.append(str(func))
                return func(*args, **(kwargs or {}))
        with Mode():
            assert torch.equal(attend(s), want)
        assert any(("shared_prefix_attention_mx" if prefix else "paged_attention_mx") in f for f in Mode.seen)
