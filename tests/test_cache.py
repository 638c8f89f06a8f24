"""Block tables, slot maps and the write into a paged cache."""
import ctypes

import pytest
import torch

from autogptq.tvm_amd import _lib, attention


def loops(lengths, counts, tables, free, tokens, block):
    """The same step, request by request and token by token, on lists."""
    tables = [list(row) for row in tables]
    width = len(tables[0]) if tables else 0
    starts, contexts, slots, positions, taken = [0], [], [], [], 0
    for b, (held, n) in enumerate(zip(lengths, counts)):
        held, n = max(held, 0), max(n, 0)
        have = -(-held // block)
        for j in range(have, -(-(held + n) // block)):
            if taken < len(free) and j < width:
                tables[b][j] = free[taken]
            elif j < width:
                tables[b][j] = None        # unspecified: whatever stood there
            taken += 1
        for p in range(held, held + n):
            j = p // block
            entry = tables[b][j] if j < width else None
            slots.append(-1 if entry is None or entry < 0 else entry * block + p % block)
            positions.append(p)
        starts.append(starts[-1] + n)
        contexts.append(held + n)
    slots += [-1] * (tokens - len(slots))
    positions += [-1] * (tokens - len(positions))
    return tables, starts, contexts, slots[:tokens], positions[:tokens], [taken]


def make(seed, B, longest, new, block, short=None, room=2):
    gen = torch.Generator().manual_seed(seed)
    lengths = torch.randint(0, longest + 1, (B,), generator=gen)
    counts = torch.randint(0, new + 1, (B,), generator=gen)
    held = (lengths + block - 1) // block
    need = (lengths + counts + block - 1) // block
    width = int(need.max()) + room if B else room
    total = int(need.sum()) + 5 if B else 5
    ids = torch.randperm(total, generator=gen)
    tables = torch.full((B, width), -1)
    at = 0
    for b in range(B):
        n = min(int(held[b]), width)
        tables[b, :n] = ids[at:at + n]
        at += n
    free = ids[at:] if short is None else ids[at:at + short]
    return lengths, counts, tables, free


CASES = [  # B, longest, new tokens at most, block, tokens beyond the sum, free blocks, table room
    (1, 0, 1, 16, 0, None, 2), (1, 37, 0, 16, 0, None, 2), (5, 40, 1, 16, 0, None, 2), (64, 4096, 1, 16, 0, None, 2),
    (7, 100, 33, 1, 0, None, 2), (300, 900, 70, 24, 0, None, 2), (3, 10, 5000, 64, 0, None, 2), (1000, 50, 3, 7, 0, None, 2),
    (6, 50, 40, 16, 9, None, 2), (6, 50, 40, 16, -5, None, 2), (6, 50, 40, 16, 0, 3, 2), (6, 50, 40, 16, 0, 0, 2),
    (6, 50, 40, 16, 0, None, -2), (0, 1, 1, 16, 4, None, 2), (8192, 3, 1, 16, 0, None, 2),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=[str(c) for c in CASES])
def test_cache_tables(case):
    B, longest, new, block, more, short, room = case
    lengths, counts, tables, free = make(31, B, longest, new, block, short, room)
    tokens = max(0, int(counts.sum()) + more)
    dev = [t.to(torch.int32).cuda() for t in (lengths, counts, tables, free)]
    for _ in range(2):      # (the table of the second call holds the entries of the first)
        made = attention.cache_tables(*dev, tokens, block)
    want = loops(lengths.tolist(), counts.tolist(), tables.tolist(), free.tolist(), tokens, block)
    assert [x.tolist() for x in made] == [list(x) for x in want[1:]]
    for got, row in zip(dev[2].tolist(), want[0]):
        assert all(e is None or g == e for g, e in zip(got, row))


@pytest.mark.gpu
def test_cache_tables_counts_negative_numbers_as_none():
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    tables = torch.full((3, 4), -1, dtype=torch.int32, device="cuda")
    made = attention.cache_tables(ints(-7, 3, 2), ints(2, -9, 1), tables, ints(5, 6, 7), 3, 2)
    assert made.starts.tolist() == [0, 2, 2, 3] and made.contexts.tolist() == [2, 3, 3]
    assert made.positions.tolist() == [0, 1, 2] and made.taken.tolist() == [2]
    assert made.slots.tolist() == [10, 11, 12] and tables[0, 0] == 5 and tables[2, 1] == 6


@pytest.mark.gpu
def test_cache_tables_writes_only_its_entries():
    wide = torch.full((2, 9), 77, dtype=torch.int32, device="cuda")
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    attention.cache_tables(ints(5, 0), ints(6, 3), wide[:, 2:6], ints(1, 2, 3, 4), 9, 4)
    assert wide.tolist() == [[77, 77, 77, 77, 1, 77, 77, 77, 77], [77, 77, 2, 77, 77, 77, 77, 77, 77]]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("layout", ["token", "head"])
@pytest.mark.parametrize("T, heads, dim, block", [(1, 1, 8, 1), (3, 2, 64, 16), (70, 8, 128, 7), (5, 3, 80, 24), (33, 1, 256, 16)])
def test_cache_write(dtype, layout, T, heads, dim, block):
    gen = torch.Generator().manual_seed(5)
    blocks = T // block + 3
    shape = (2, blocks, block, heads, dim) if layout == "token" else (2, blocks, heads, block, dim)
    cache = torch.randn(shape, generator=gen).to(dtype).cuda()
    cache = cache if layout == "token" else cache.transpose(2, 3)
    slots = torch.randperm(blocks * block, generator=gen)[:T].to(torch.int32)
    slots[T // 2] = -1 if T > 1 else slots[T // 2]
    if T > 4:
        slots[1], slots[3] = blocks * block, 2 ** 31 - 1        # outside of the cache
    wide = torch.randn((T, 3 * heads * dim), generator=gen).to(dtype).cuda()
    forms = {"columns": [wide[:, i * heads * dim:(i + 1) * heads * dim].view(T, heads, dim) for i in (1, 2)],
             "odd offset": [torch.cat([wide.new_zeros(1), wide[:, :heads * dim].reshape(-1)])[1:].view(T, heads, dim)] * 2,
             "heads first": [wide[:, :heads * dim].reshape(T, heads, dim).transpose(0, 1).contiguous().transpose(0, 1)] * 2}
    for name, (k, v) in forms.items():
        want = cache.clone()
        for t, s in enumerate(slots.tolist()):
            if 0 <= s < blocks * block:
                want[0][s // block, s % block], want[1][s // block, s % block] = k[t], v[t]
        got = cache.clone()
        attention.cache_write(k, v, got[0], got[1], slots.cuda())
        assert torch.equal(got, want), name


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    cache = torch.zeros(2, 4, 16, 2, 64, device="cuda", dtype=torch.float16)
    k = torch.zeros(3, 2, 64, device="cuda", dtype=torch.float16)
    slots = torch.arange(3, dtype=torch.int32, device="cuda")
    write = lambda k=k, v=k, kc=cache[0], vc=cache[1], s=slots: attention.cache_write(k, v, kc, vc, s)
    write()
    for call, text in ((lambda: write(k=k.bfloat16()), "the cache"), (lambda: write(k=k[:, :1]), r"\[tokens, 2, 64\]"),
                       (lambda: write(v=k[:2]), "v 2"), (lambda: write(s=slots[:2]), "vector of 3"),
                       (lambda: write(s=slots.long()), "int32"), (lambda: write(vc=cache[1].cpu()), "no CPU fallback"),
                       (lambda: write(k=k.clone().requires_grad_()), "no backward"),
                       (lambda: write(kc=cache[0][..., :60], vc=cache[1][..., :60]), "multiple of 8")):
        with pytest.raises(RuntimeError, match=text):
            call()
    write(k=k[:0], v=k[:0], s=slots[:0])
    ints = torch.ones(3, dtype=torch.int32, device="cuda")
    tables = torch.zeros(3, 4, dtype=torch.int32, device="cuda")
    for args, text in (((ints.float(), ints, tables, ints, 3, 16), "int32"), ((ints, ints[:2], tables, ints, 3, 16), "vector of 3"),
                       ((ints, ints, tables[:2], ints, 3, 16), "width"), ((ints, ints, tables, ints, -1, 16), "tokens"),
                       ((ints, ints, tables, ints, 3, 0), "block_size"), ((ints, ints, tables.cpu(), ints, 3, 16), "no CPU fallback")):
        with pytest.raises(RuntimeError, match=text):
            attention.cache_tables(*args)
    many = torch.zeros(8193, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="at most 8192"):
        attention.cache_tables(many, many, torch.zeros(8193, 1, dtype=torch.int32, device="cuda"), ints, 0, 16)


def test_the_entry_points_refuse():
    lib, p = _lib.lib(), 0x1000
    tables = lambda lengths=p, stride=4, width=4, free=p, n_free=3, B=2, T=3, block=16, starts=p, slots=p: \
        lib.gptq_hip_cache_tables(lengths, p, p, stride, width, free, n_free, B, T, block, starts, p, slots, p, p, None)
    for more, status in ((dict(lengths=None), _lib.ERR_BAD_ARG), (dict(stride=3), _lib.ERR_BAD_ARG), (dict(width=-1), _lib.ERR_BAD_ARG),
                         (dict(free=None), _lib.ERR_BAD_ARG), (dict(B=-1), _lib.ERR_BAD_ARG), (dict(T=-1), _lib.ERR_BAD_ARG),
                         (dict(block=0), _lib.ERR_BAD_ARG), (dict(starts=None), _lib.ERR_BAD_ARG), (dict(slots=None), _lib.ERR_BAD_ARG),
                         (dict(B=8193), _lib.ERR_UNSUPPORTED)):
        assert tables(**more) == status, more
    cache = _lib.Cache(k=p, v=p, type=0, blocks=4, block_size=16, heads=2, dim=64, block_stride=2048, slot_stride=128, head_stride=64)
    write = lambda c=cache, k=p, strides=(128, 64, 128, 64), slots=p, T=3: \
        lib.gptq_hip_cache_write(None if c is None else ctypes.byref(c), k, p, *strides, slots, T, None)
    for more in (dict(c=None), dict(k=None), dict(k=0x1004), dict(strides=(128, 64, 130, 64)), dict(slots=None), dict(T=-1)):
        assert write(**more) == _lib.ERR_BAD_ARG, more
    assert write(T=0) == _lib.OK


@pytest.mark.gpu
def test_what_is_written_counts_as_written():
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    for call in (attention.cache_tables, torch.ops.gptq_hip.cache_tables):
        tables = torch.full((2, 4), -1, dtype=torch.int32, device="cuda")
        before = tables._version
        call(ints(0, 3), ints(2, 2), tables, ints(5, 6, 7), 4, 2)
        assert tables._version > before, call
    with torch.inference_mode():
        tables = torch.full((2, 4), -1, dtype=torch.int32, device="cuda")
        attention.cache_tables(ints(0, 3), ints(2, 2), tables, ints(5, 6, 7), 4, 2)
    for call in (attention.cache_write, torch.ops.gptq_hip.cache_write):
        cache = torch.zeros(2, 4, 16, 2, 64, device="cuda", dtype=torch.float16)
        k, v = torch.ones(2, 3, 2, 64, device="cuda", dtype=torch.float16)
        before = cache._version
        call(k, v, cache[0], cache[1], ints(0, 1, 2))
        assert cache._version > before, call


# above 32768 tokens a thread takes four neighbours: sums that leave a remainder, room beyond and below them, requests without tokens,
# blocks of one and of no power of two, too few free blocks, too narrow tables
LARGE = [  # as CASES, and every how many requests have none
    (5, 300, 20000, 16, 0, None, 2, 0), (400, 900, 500, 24, 3, None, 2, 3), (400, 900, 500, 7, -2, None, 2, 2), (3000, 5, 30, 1, 1, None, 2, 5),
    (9, 100, 15000, 64, -30001, None, 2, 0), (1, 7, 70001, 16, 2, None, 2, 0), (40, 50, 3000, 16, 50000, 1000, 2, 4),
    (40, 50, 3000, 16, 0, None, -9, 4), (8192, 3, 12, 16, 0, None, 2, 7), (2, 0, 1, 16, 40001, None, 2, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", LARGE, ids=[str(c) for c in LARGE])
def test_cache_tables_of_many_tokens(case):
    B, longest, new, block, more, short, room, every = case
    lengths, counts, tables, free = make(32, B, longest, new, block, short, room)
    if every:
        counts[::every] = 0
    if B == 1:
        counts[0] = new
    tokens = int(counts.sum()) + more
    assert tokens > 32768
    dev = [t.to(torch.int32).cuda() for t in (lengths, counts, tables, free)]
    for _ in range(2):
        torch.full((tokens + 20000,), 77, dtype=torch.int32, device="cuda")      # what the results' memory holds
        made = attention.cache_tables(*dev, tokens, block)
    want = loops(lengths.tolist(), counts.tolist(), tables.tolist(), free.tolist(), tokens, block)
    assert [x.tolist() for x in made] == [list(x) for x in want[1:]]
    for got, row in zip(dev[2].tolist(), want[0]):
        assert all(e is None or g == e for g, e in zip(got, row))
