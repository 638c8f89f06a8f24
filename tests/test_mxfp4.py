"""A cache in MXFP4: the write that quantises and the read, against the format's definition in 64 bits."""
import ctypes

import pytest
import torch

from autogptq.tvm_amd import _lib, attention
from autogptq.tvm_amd.attention import Mxfp4
from tests.mxfp4_util import EXPONENTS, VALUES, decode, empty, encode, widths

HALF, BF16 = torch.float16, torch.bfloat16
ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")


def clone(cache):
    return Mxfp4(*(t.clone(memory_format=torch.preserve_format) for t in cache))


def test_the_definition():
    """The oracle itself, on numbers that were worked out by hand."""
    x = torch.tensor([[0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0] + [0.0] * 8 + [-0.25, -0.75, -1.3, 6.9] + [0.0] * 12], dtype=HALF)
    codes, scales = encode(x)
    assert scales.tolist() == [[127]]
    assert codes[0, :4].tolist() == [0x20, 0x42, 0x64, 0x76] and codes[0, 8:10].tolist() == [0xA8, 0x7B]
    assert encode(torch.full((1, 32), 7.0, dtype=HALF))[1].tolist() == [[128]]          # 1.75 x 4: the next exponent
    assert encode(torch.full((1, 32), 6.996, dtype=HALF))[1].tolist() == [[127]]
    assert encode(torch.full((1, 8), 65504.0, dtype=HALF))[1].tolist() == [[140]]
    assert encode(torch.full((1, 8), 2.0 ** -24, dtype=HALF))[1].tolist() == [[104]]
    assert encode(torch.full((1, 8), 3e38, dtype=BF16))[1].tolist() == [[252]]
    assert encode(torch.zeros((1, 40), dtype=BF16))[1].tolist() == [[2, 2]]
    assert decode(*encode(torch.full((1, 8), float("inf"), dtype=HALF)), 8).isnan().all()
    d = decode(codes, scales, 32)
    assert d[0, :8].tolist() == [0, 1, 1, 2, 2, 4, 4, 6] and d[0, 16:20].tolist() == [0, -1, -1.5, 6]


def rows(seed, T, heads, dim, dtype):
    """Rows of very different sizes, some of them zero, with zeros and with numbers between two codes among them."""
    gen = torch.Generator().manual_seed(seed)
    low, high = (-18, 10) if dtype == HALF else (-60, 60)
    x = torch.randn(T, heads, dim, generator=gen)
    x *= torch.exp2(torch.randint(low, high, (T, heads, 1), generator=gen).float())
    x[..., ::29] *= 4
    x[torch.rand(T, heads, dim, generator=gen) < 0.05] = 0
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -6.0])
    x[T // 2, 0, :8] = ties
    x[T - 1, heads - 1] = 0
    return x.to(dtype)


WRITES = [(1, 1, 8, 1), (3, 2, 64, 16), (70, 8, 128, 7), (5, 3, 80, 24), (33, 1, 256, 16), (9, 2, 72, 16), (40, 2, 96, 16), (11, 3, 136, 8),
          (6, 1, 32, 4), (7, 2, 200, 5)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [HALF, BF16])
@pytest.mark.parametrize("layout", ["token", "head"])
@pytest.mark.parametrize("T, heads, dim, block", WRITES)
def test_write(dtype, layout, T, heads, dim, block):
    gen = torch.Generator().manual_seed(5)
    blocks = T // block + 3
    slots = torch.randperm(blocks * block, generator=gen)[:T].to(torch.int32)
    slots[T // 2] = -1 if T > 5 else slots[T // 2]
    if T > 4:
        slots[1], slots[3] = blocks * block, 2 ** 31 - 1        # outside of the cache
    wide = torch.cat([rows(i, T, heads, dim, dtype).reshape(T, heads * dim) for i in (1, 2, 3)], 1).cuda()
    forms = {"columns": [wide[:, i * heads * dim:(i + 1) * heads * dim].view(T, heads, dim) for i in (1, 2)],
             "odd offset": [torch.cat([wide.new_zeros(1), wide[:, :heads * dim].reshape(-1)])[1:].view(T, heads, dim)] * 2,
             "heads first": [wide[:, :heads * dim].reshape(T, heads, dim).transpose(0, 1).contiguous().transpose(0, 1)] * 2}
    groups = -(-dim // 32)
    for name, (k, v) in forms.items():
        got = empty(blocks, block, heads, dim, layout)
        want = [clone(c) for c in got]
        for x, c in zip((k, v), want):
            codes, scales = encode(x)
            for t, s in enumerate(slots.tolist()):
                if 0 <= s < blocks * block:
                    c.codes[s // block, s % block], c.scales[s // block, s % block, :, :groups] = codes[t], scales[t]
        attention.cache_write(k, v, *got, slots.cuda())
        for g, w in zip(got, want):
            assert torch.equal(g.scales[..., :groups], w.scales[..., :groups]), name
            assert torch.equal(g.codes, w.codes), name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [HALF, BF16])
def test_write_of_every_number(dtype):
    """All 2^16 patterns (infinities and NaN among them) as a group's largest number and as one beside larger ones."""
    bits = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(dtype)
    T = 1 << 16
    k = torch.zeros(T, 1, 64, dtype=dtype)
    k[:, 0, 5] = bits
    shift = torch.arange(64)
    k[:, 0, 32:] = torch.where(shift[:32] % 2 == 0, bits[:, None], bits.flip(0)[:, None])
    v = bits[torch.randperm(T, generator=torch.Generator().manual_seed(1))].view(-1, 1, 64)
    v = torch.cat([v] * 64)
    cache = empty(T // 64, 64, 1, 64)
    attention.cache_write(k.cuda(), v.cuda(), *cache, torch.arange(T, dtype=torch.int32, device="cuda"))
    for x, c in zip((k, v), cache):
        codes, scales = encode(x)
        assert torch.equal(c.scales.flatten(0, 1).cpu(), scales)
        assert torch.equal(c.codes.flatten(0, 1).cpu(), codes)
    # what finite groups stand for is a value of the type, and is what comes back
    back = attention.cache_read(*cache, torch.arange(T, dtype=torch.int32, device="cuda"), 64, dtype)
    for x, b in zip((k, v), back):
        want = decode(*encode(x), 64)
        assert torch.equal(want.to(dtype).double().nan_to_num(7e77), want.nan_to_num(7e77))
        assert torch.equal(b.cpu().double().nan_to_num(7e77), want.nan_to_num(7e77))


@pytest.mark.gpu
def test_the_error_of_a_write():
    """Half a step of the codes: 1/4 of 2^e below 2 (1/8 of the group's largest magnitude), 1/2 below 4, 1 up to 7."""
    for dtype in (HALF, BF16):
        x = torch.randn(500, 2, 128, generator=torch.Generator().manual_seed(2)).to(dtype)
        cache = empty(500, 1, 2, 128)
        slots = torch.arange(500, dtype=torch.int32, device="cuda")
        attention.cache_write(x.cuda(), x.cuda(), *cache, slots)
        back = attention.cache_read(*cache, slots, 128, dtype)[0].cpu().double()
        most = x.double().unflatten(-1, (4, 32)).abs().amax(-1, keepdim=True)
        err = (back - x.double()).unflatten(-1, (4, 32)).abs()
        assert bool((err <= most / 3.5).all()) and bool((err <= torch.maximum(most / 14, x.double().unflatten(-1, (4, 32)).abs() / 4)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["token", "head"])
@pytest.mark.parametrize("T, heads, dim, block", WRITES)
def test_read(layout, T, heads, dim, block):
    gen = torch.Generator().manual_seed(6)
    blocks = T // block + 3
    cache = empty(blocks, block, heads, dim, layout)
    slots = torch.randint(0, blocks * block, (T,), generator=gen).to(torch.int32)      # (some of them twice)
    if T > 4:
        slots[0], slots[2], slots[3] = -1, blocks * block, 2 ** 31 - 1
    inside = [t for t, s in enumerate(slots.tolist()) if 0 <= s < blocks * block]
    at = slots[inside].long()
    for dtype in (HALF, BF16):
        for c in cache:
            c.codes.copy_(torch.randint(0, 256, c.codes.shape, generator=gen))
            low, high = EXPONENTS[dtype]
            c.scales.copy_(torch.randint(low + 127, high + 128, c.scales.shape, generator=gen))
            c.scales[blocks - 1, block - 1] = 255
        for got, c in zip(attention.cache_read(*cache, slots.cuda(), dim, dtype), cache):
            want = torch.zeros(T, heads, dim, dtype=torch.float64)
            want[inside] = decode(c.codes.cpu()[at // block, at % block], c.scales.cpu()[at // block, at % block], dim)
            assert got.shape == want.shape and got.dtype == dtype
            assert torch.equal(got.cpu().double().nan_to_num(7e77), want.nan_to_num(7e77))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [HALF, BF16])
@pytest.mark.parametrize("layout", ["token", "head"])
def test_read_of_other_caches(dtype, layout):
    gen = torch.Generator().manual_seed(7)
    shape = (2, 5, 7, 3, 40) if layout == "token" else (2, 5, 3, 7, 40)
    cache = torch.randn(shape, generator=gen).to(dtype).cuda()
    cache = cache if layout == "token" else cache.transpose(2, 3)
    slots = ints(0, 34, -1, 13, 13, 35, 20)
    for got, c in zip(attention.cache_read(cache[0], cache[1], slots), cache):
        want = torch.stack([c[s // 7, s % 7] if 0 <= s < 35 else torch.zeros_like(c[0, 0]) for s in slots.tolist()])
        assert torch.equal(got, want)
    assert attention.cache_read(cache[0], cache[1], slots[:0])[0].shape == (0, 3, 40)
    for more in (dict(dim=32), dict(dtype=torch.float32)):
        with pytest.raises(ValueError, match="rows of 40"):
            attention.cache_read(cache[0], cache[1], slots, **more)


@pytest.mark.gpu
def test_defaults_of_a_read():
    cache = empty(2, 4, 1, 80)
    k = torch.randn(3, 1, 80, device="cuda").half()
    attention.cache_write(k, -k, *cache, ints(0, 5, 2))
    got, minus = attention.cache_read(*cache, ints(0, 5, 2))
    assert got.shape == (3, 1, 96) and got.dtype == HALF and bool((got[..., 80:] == 0).all())
    assert torch.equal(got[..., :80], attention.cache_read(*cache, ints(0, 5, 2), 80)[0]) and torch.equal(got[..., :80], -minus[..., :80])


@pytest.mark.gpu
def test_offsets_past_32_bits():
    blocks = (1 << 32) // (16 * 64) + 100
    cache = attention.mxfp4_cache(blocks, 16, 1, 128)
    slots = ints(blocks * 16 - 1, (blocks - 5) * 16 + 2, 3)
    k, v = torch.randn(2, 3, 1, 128, device="cuda").half()
    attention.cache_write(k, v, *cache, slots)
    for got, x in zip(attention.cache_read(*cache, slots, 128), (k, v)):
        assert torch.equal(got.double(), decode(*encode(x), 128))


@pytest.mark.gpu
def test_on_another_stream_and_captured():
    cache = empty(30, 16, 2, 128)
    k, v = torch.randn(2, 300, 2, 128, device="cuda").half()
    slots = torch.randperm(480, generator=torch.Generator().manual_seed(3))[:300].to(torch.int32).cuda()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()

    def both():
        attention.cache_write(k, v, *cache, slots)
        return attention.cache_read(*cache, slots, 128)
    with torch.cuda.stream(side):
        want = both()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = both()
        for i in range(3):
            k.mul_(-1)
            for c in cache:
                c.codes.fill_(0x11)
            graph.replay()
            side.synchronize()
            eager = both()
            assert torch.equal(got[0], want[0] if i % 2 else -want[0]) and torch.equal(got[1], want[1])
            assert all(torch.equal(e, g) for e, g in zip(eager, got))
            side.synchronize()


def test_cpu_tensors_and_mixed_caches_are_refused():
    cache = empty(2, 16, 1, 64, device="cpu")
    k = torch.zeros(3, 1, 64, dtype=HALF)
    slots = torch.arange(3, dtype=torch.int32)
    for call in (lambda: attention.cache_write(k, k, *cache, slots), lambda: attention.cache_read(*cache, slots, 64),
                 lambda: attention.cache_read(k[:, None], k[:, None], slots)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()
    with pytest.raises(TypeError, match="both be"):
        attention.cache_write(k, k, cache[0], k[:, None], slots)
    with pytest.raises(TypeError, match="both be"):
        attention.cache_read(k[:, None], cache[1], slots)
    for dim in (0, 4, 100, 264):
        with pytest.raises(ValueError, match="multiple of 8"):
            attention.mxfp4_cache(2, 16, 1, dim, device="cpu")
    for dim, shapes in ((8, (16, 2)), (80, (48, 4)), (128, (64, 4)), (136, (80, 8))):
        made = attention.mxfp4_cache(3, 5, 2, dim, device="cpu")
        assert [tuple(t.shape) for c in made for t in c] == 2 * [(3, 5, 2, n) for n in shapes] and widths(dim) == shapes


def test_meta_tensors_have_a_shape():
    cache = [Mxfp4(*(t.to("meta") for t in c)) for c in empty(2, 16, 3, 80, device="cpu")]
    k = torch.zeros(4, 3, 80, dtype=BF16, device="meta")
    slots = torch.zeros(4, dtype=torch.int32, device="meta")
    assert attention.cache_write(k, k, *cache, slots) is None
    for out in (attention.cache_read(*cache, slots, 80, BF16), attention.cache_read(k[:, None], k[:, None], slots)):
        assert [(t.device.type, t.shape, t.dtype) for t in out] == 2 * [("meta", (4, 3, 80), BF16)]


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    cache = empty(4, 16, 2, 64)
    k = torch.zeros(3, 2, 64, device="cuda", dtype=HALF)
    slots = ints(0, 1, 2)
    write = lambda k=k, v=k, kc=cache[0], vc=cache[1], s=slots: attention.cache_write(k, v, kc, vc, s)
    write()
    swap = lambda c, **more: c._replace(**more)
    token = empty(4, 16, 2, 64, "token")
    for call, text in ((lambda: write(k=k.float(), v=k.float()), "float16 or bfloat16"), (lambda: write(v=k.bfloat16()), "v is"),
                       (lambda: write(k=k[:, :1]), r"\[tokens, 2, 64\]"), (lambda: write(k=k[..., :32]), "uint8|k_codes must be|must be"),
                       (lambda: write(v=k[:2]), "v 2"), (lambda: write(s=slots[:2]), "vector of 3"), (lambda: write(s=slots.long()), "int32"),
                       (lambda: write(kc=swap(cache[0], codes=cache[0].codes.cpu())), "no CPU fallback"),
                       (lambda: write(vc=swap(cache[1], scales=cache[1].scales.cpu())), "no CPU fallback"),
                       (lambda: write(kc=swap(cache[0], codes=cache[0].codes.to(torch.int8))), "uint8"),
                       (lambda: write(kc=swap(cache[0], scales=cache[0].scales[..., :1])), "k_scales must be"),
                       (lambda: write(kc=swap(cache[0], scales=cache[0].scales[:3])), "same"),
                       (lambda: write(kc=swap(cache[0], scales=cache[0].scales[:3]), vc=swap(cache[1], scales=cache[1].scales[:3])), "same rows"),
                       (lambda: write(vc=token[1]), "same shapes and strides"), (lambda: write(k=k.clone().requires_grad_()), "no backward"),
                       (lambda: write(k=k[:0].view(0, 2, 64)[:, :, :60], v=k[:0]), "multiple of 8"),
                       (lambda: attention.cache_read(*cache, slots, 80), "k_codes must be"),
                       (lambda: attention.cache_read(*cache, slots, 64, torch.float32), "float16 or bfloat16"),
                       (lambda: attention.cache_read(*cache, slots.long(), 64), "int32")):
        with pytest.raises(RuntimeError, match=text):
            call()
    write(k=k[:0], v=k[:0], s=slots[:0])
    assert attention.cache_read(*cache, slots[:0], 64)[0].shape == (0, 2, 64)
    # rows that are not where 16-byte loads reach them
    raw = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda")
    odd = raw[8:8 + 4 * 16 * 2 * 32].view(4, 16, 2, 32)
    with pytest.raises(RuntimeError, match="16-byte aligned"):
        write(kc=swap(cache[0], codes=odd), vc=swap(cache[1], codes=odd))
    odd = raw[1:1 + 4 * 16 * 2 * 2].view(4, 16, 2, 2)
    with pytest.raises(RuntimeError, match="2-byte aligned"):
        write(kc=swap(cache[0], scales=odd), vc=swap(cache[1], scales=odd))


def test_the_entry_points_refuse():
    lib, p = _lib.lib(), 0x1000

    def cache(**more):
        c = dict(k=p, v=p, k_scales=p, v_scales=p, type=0, blocks=4, block_size=16, heads=2, dim=128, block_stride=2048, slot_stride=128,
                 head_stride=64, scale_block_stride=128, scale_slot_stride=8, scale_head_stride=4)
        return _lib.CacheMx(**{**c, **more})
    write = lambda c, k=p, strides=(128, 64, 128, 64), slots=p, T=3: lib.gptq_hip_cache_write_mx(ctypes.byref(c), k, p, *strides, slots, T, None)
    read = lambda c, k=p, v=p, slots=p, T=3: lib.gptq_hip_cache_read_mx(ctypes.byref(c), slots, T, k, v, None)
    for more, status in ((dict(k=None), _lib.ERR_BAD_ARG), (dict(v=p + 8), _lib.ERR_BAD_ARG), (dict(k_scales=None), _lib.ERR_BAD_ARG),
                         (dict(v_scales=p + 2), _lib.ERR_BAD_ARG), (dict(type=2), _lib.ERR_BAD_ARG), (dict(blocks=0), _lib.ERR_BAD_ARG),
                         (dict(block_size=0), _lib.ERR_BAD_ARG), (dict(heads=0), _lib.ERR_BAD_ARG), (dict(dim=100), _lib.ERR_BAD_ARG),
                         (dict(dim=264), _lib.ERR_UNSUPPORTED), (dict(block_stride=2056), _lib.ERR_BAD_ARG), (dict(slot_stride=-16), _lib.ERR_BAD_ARG),
                         (dict(scale_slot_stride=2), _lib.ERR_BAD_ARG), (dict(blocks=1 << 27), _lib.ERR_UNSUPPORTED),
                         (dict(blocks=1 << 20, block_stride=1 << 20), _lib.ERR_UNSUPPORTED),
                         (dict(blocks=1 << 20, scale_block_stride=1 << 20), _lib.ERR_UNSUPPORTED)):
        assert write(cache(**more), T=0) == status and read(cache(**more), T=0) == status, more
    c = cache()
    for got in (write(c, k=None), write(c, k=p + 4), write(c, strides=(128, 64, 130, 64)), write(c, slots=None), write(c, T=-1), read(c, k=None),
                read(c, v=p + 4), read(c, slots=None), read(c, T=-1), lib.gptq_hip_cache_write_mx(None, p, p, 8, 8, 8, 8, p, 1, None),
                lib.gptq_hip_cache_read_mx(None, p, 1, p, p, None), lib.gptq_hip_cache_read(None, p, 1, p, p, None)):
        assert got == _lib.ERR_BAD_ARG
    assert write(c, T=0) == _lib.OK and read(c, T=0) == _lib.OK
    plain = _lib.Cache(k=p, v=p, type=0, blocks=4, block_size=16, heads=2, dim=64, block_stride=2048, slot_stride=128, head_stride=64)
    for args in ((None, 3, p, p), (p, -1, p, p), (p, 3, None, p), (p, 3, p, p + 4)):
        assert lib.gptq_hip_cache_read(ctypes.byref(plain), *args, None) == _lib.ERR_BAD_ARG
    assert lib.gptq_hip_cache_read(ctypes.byref(plain), None, 0, None, None, None) == _lib.OK


@pytest.mark.gpu
def test_through_the_dispatcher():
    from torch.overrides import TorchFunctionMode

    cache = empty(4, 16, 2, 64)
    k, v = torch.randn(2, 3, 2, 64, device="cuda").half()
    slots = ints(0, 9, 2)
    attention.cache_write(k, v, *cache, slots)
    want = attention.cache_read(*cache, slots, 64)
    other = empty(4, 16, 2, 64)
    flat = [t for c in other for t in c]
    before = [t._version for t in flat]
    torch.ops.gptq_hip.cache_write_mx(k, v, *flat, slots)
    assert all(t._version > b for t, b in zip(flat, before))
    before = [t._version for t in flat]
    attention.cache_write(k, v, *other, slots)
    assert all(t._version > b for t, b in zip(flat, before))
    assert all(torch.equal(a, b) for a, b in zip(torch.ops.gptq_hip.cache_read_mx(*flat, slots, 64, HALF), want))
    assert all(torch.equal(a, b) for c, d in zip(cache, other) for a, b in zip(c, d))

    class Mode(TorchFunctionMode):
        seen = []

        def __torch_function__(self, func, types, args=(), kwargs=None):
            self.seen.append(str(func))
            return func(*args, **(kwargs or {}))
    with Mode():
        attention.cache_write(k, v, *other, slots)
        got = attention.cache_read(*other, slots, 64)
        attention.cache_read(k[:, None], v[:, None], slots)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for name in ("cache_write_mx", "cache_read_mx", "cache_read"):
        assert any(name in f for f in Mode.seen), (name, Mode.seen)
    with torch.inference_mode():
        made = empty(4, 16, 2, 64)
        attention.cache_write(k, v, *made, slots)
    assert all(torch.equal(a, b) for a, b in zip(attention.cache_read(*made, slots, 64), want))


@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [True, False])
def test_read_of_more_than_the_caches_hold(quantised):
    gen = torch.Generator(device="cuda").manual_seed(9)
    rand = lambda shape: torch.randint(0, 256, shape, dtype=torch.uint8, device="cuda", generator=gen)
    if quantised:
        cache = attention.mxfp4_cache(300, 64, 4, 128)
        for c in cache:
            c.codes.copy_(rand(c.codes.shape))
            c.scales.copy_(rand(c.scales.shape) % 20 + 117)
    else:
        cache = torch.randn(2, 300, 64, 4, 128, device="cuda", generator=gen).half().unbind()
    slots = torch.randint(-50, 300 * 64 + 50, (17001,), device="cuda", generator=gen, dtype=torch.int32)
    inside = (slots >= 0) & (slots < 300 * 64)
    at = torch.where(inside, slots, 0).long()
    for got, c in zip(attention.cache_read(*cache, slots, 128), cache):
        want = decode(c.codes[at // 64, at % 64], c.scales[at // 64, at % 64], 128) if quantised else c[at // 64, at % 64].double()
        assert torch.equal(got.double(), torch.where(inside[:, None, None], want, 0.0))
