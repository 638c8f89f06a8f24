"""``PagedCache``: the host's bookkeeping, and a small decoder served from it."""
import os
import sys

import pytest
import torch

from autogptq.tvm_amd import PagedCache

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.gpu
def test_a_decoder_is_served_from_it():
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    try:
        import serve_paged
    finally:
        sys.path.pop(0)
    # (half-precision rounding through two layers of products and normalisations; the example asserts 2e-2 at every step)
    assert serve_paged.main(verbose=False) < 2e-2


def cache(**more):
    return PagedCache(**{**dict(layers=1, blocks=12, block_size=4, kv_heads=1, dim=8, max_requests=3, max_context=24), **more})


@pytest.mark.gpu
def test_blocks_are_dealt_out_and_come_back():
    c = cache()
    s = c.step([0, 2], [5, 3])
    assert c.free_blocks == 9 and (c.length(0), c.length(1), c.length(2)) == (5, 0, 3)
    assert s.positions.tolist() == [0, 1, 2, 3, 4, 0, 1, 2] and s.contexts.tolist() == [5, 3] and s.max_context == 5
    s = c.step([2, 0, 1], [2, 0, 1])        # another order, and a request that gets nothing
    assert c.free_blocks == 7 and s.contexts.tolist() == [5, 5, 1] and s.starts.tolist() == [0, 2, 2, 3]
    used = [e for e in c.tables.flatten().tolist() if e >= 0]
    assert len(used) == len(set(used)) == 5
    assert s.slots.tolist()[:2] == [int(c.tables[2, 0]) * 4 + 3, int(c.tables[2, 1]) * 4]
    c.free(0)
    c.free(1)
    assert c.free_blocks == 10 and c.length(0) == 0
    c.step([0], [24])
    with pytest.raises(RuntimeError, match="does not fit"):
        c.step([0], [1])
    c.step([1], [12])
    before = c.tables.clone()
    with pytest.raises(RuntimeError, match="2 blocks are needed and 1 are free"):
        c.step([2], [9])
    assert torch.equal(c.tables, before) and c.length(2) == 5
    c.free(0), c.free(1), c.free(2)
    assert sorted(c._free.tolist()) == list(range(12))


@pytest.mark.gpu
def test_trim_gives_back_what_the_window_has_left():
    c = cache()
    c.step([1], [20])
    assert c.trim(1, window=6, sinks=1) == 2            # tokens up to 14 are unseen from token 20 on: blocks 1 and 2
    assert c.tables[1].tolist()[1:3] == [-1, -1] and c.free_blocks == 9
    assert c.trim(1, window=6, sinks=1) == 0
    c.step([1], [4])
    assert c.trim(1, window=6, sinks=1) == 1 and c.free_blocks == 9
    c.free(1)
    assert sorted(c._free.tolist()) == list(range(12))


@pytest.mark.gpu
def test_shared_prefixes():
    c = cache()
    c.step([0], [6])
    c.share(0, 1)
    s = c.step([1], [3])
    assert s.prefix[1] == 6 and s.prefix[0].tolist() == c.tables[0, :2].tolist() and s.positions.tolist() == [6, 7, 8]
    with pytest.raises(ValueError, match="one prefix"):
        c.step([1, 2], [1, 1])
    with pytest.raises(ValueError, match="has tokens"):
        c.share(0, 1)
    with pytest.raises(ValueError, match="behind a prefix itself"):
        c.share(1, 2)
    c.share(0, 2)
    assert c.step([1, 2], [1, 2]).prefix[1] == 6
    q = torch.zeros(3, 1, 8, dtype=torch.float16, device="cuda")
    with pytest.raises(NotImplementedError):
        c.attend(0, q, c.step([1, 2], [1, 2]), window=4)


def test_refusals():
    c = cache(device="cpu")
    with pytest.raises(ValueError, match="distinct"):
        c.step([1, 1], [1, 1])
    with pytest.raises(ValueError, match="at least 0"):
        c.step([1], [-1])
    with pytest.raises(RuntimeError, match="does not fit"):
        c.step([1], [25])
    with pytest.raises(ValueError, match="window"):
        c.trim(0, 0)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        c.step([1], [3])


@pytest.fixture
def host(monkeypatch):
    """The bookkeeping without a GPU: cache_tables request by request, on CPU tensors."""
    from autogptq.tvm_amd import attention

    def cache_tables(lengths, counts, tables, free, tokens, block):
        taken, slots, positions, starts = 0, [], [], [0]
        for b, (held, n) in enumerate(zip(lengths.tolist(), counts.tolist())):
            for p in range(held, held + n):
                if p % block == 0:
                    tables[b, p // block] = free[taken]
                    taken += 1
                slots.append(int(tables[b, p // block]) * block + p % block)
                positions.append(p)
            starts.append(starts[-1] + n)
        ints = lambda x: torch.tensor(x, dtype=torch.int32)
        return attention.CacheTables(ints(starts), lengths + counts, ints(slots), ints(positions), ints([taken]))
    monkeypatch.setattr(attention, "cache_tables", cache_tables)
    return lambda **more: cache(device="cpu", **more)


def test_a_source_stays_while_others_stand_behind_it(host):
    c = host(max_requests=4)
    c.step([0], [6])
    c.share(0, 1)
    c.share(0, 2)
    c.step([1], [3])
    blocks = c.tables[0, :2].tolist()
    for call in (lambda: c.free(0), lambda: c.trim(0, 1)):
        with pytest.raises(ValueError, match=r"\[1, 2\] stand behind"):
            call()
    assert c.tables[0, :2].tolist() == blocks and c.length(0) == 6
    c.free(1)
    with pytest.raises(ValueError, match=r"\[2\] stand behind"):
        c.free(0)
    # a request that ended stands behind nobody, whatever it gets next
    c.step([1], [4])
    assert c.step([2], [1]).prefix[0].tolist() == blocks
    c.free(2)
    c.free(0)
    c.free(1)
    assert sorted(c._free.tolist()) == list(range(12))


def test_a_source_may_go_on(host):
    c = host()
    c.step([0], [6])
    c.share(0, 1)
    blocks = c.tables[0, :2].tolist()
    c.step([0], [7])
    assert c.step([1], [2]).prefix[0].tolist() == blocks and c.step([1], [1]).prefix[1] == 6
    c.share(0, 2)
    with pytest.raises(ValueError, match="one prefix"):       # (13 tokens, not 6)
        c.step([1, 2], [1, 1])
    assert c.step([2], [1]).prefix[1] == 13


def test_a_request_behind_a_prefix_is_not_trimmed(host):
    c = host()
    c.step([0], [6])
    c.share(0, 1)
    c.step([1], [12])
    with pytest.raises(NotImplementedError):
        c.trim(1, 4)
    assert -1 not in c.tables[1, :3].tolist()


@pytest.mark.gpu
def test_a_source_that_goes_on_is_not_seen():
    """(The prefix ends within a block, which the source fills up.)"""
    c = cache(dim=64, blocks=40, max_context=80)
    gen = torch.Generator().manual_seed(3)
    draw = lambda n: torch.randn(2, n, 1, 64, generator=gen).half().cuda()
    c.write(0, *draw(38), c.step([0], [38]))
    c.share(0, 1)
    s = c.step([1], [3])
    k, v = draw(3)
    c.write(0, k, v, s)
    q = torch.randn(3, 1, 64, generator=gen).half().cuda()
    want = c.attend(0, q, s)
    k, v = draw(9)
    c.write(0, torch.full_like(k, float("nan")), torch.full_like(v, float("nan")), c.step([0], [9]))
    assert bool(want.isfinite().all()) and torch.equal(c.attend(0, q, s), want)


def test_a_second_trim_with_other_sinks_loses_no_blocks(host):
    c = host(blocks=40, max_context=160)
    c.step([0], [100])
    assert c.trim(0, window=40, sinks=1) == 14                 # blocks 1 to 14
    with pytest.raises(ValueError, match="60 sinks are too many"):
        c.trim(0, window=8, sinks=60)
    assert c.trim(0, window=8, sinks=4) == 8 and c.trim(0, window=200, sinks=0) == 0
    c.step([0], [20])
    assert c.trim(0, window=8, sinks=0) == 5
    c.free(0)
    assert sorted(c._free.tolist()) == list(range(40))
    c.step([1], [100])
    assert c.trim(1, window=40, sinks=8) == 13 and c.trim(1, window=8, sinks=1) == 8
    c.free(1)
    assert sorted(c._free.tolist()) == list(range(40))


def test_blocks_that_were_given_back_are_not_read(host, monkeypatch):
    from autogptq.tvm_amd import attention

    seen = []
    monkeypatch.setattr(attention, "paged_attention", lambda *args, window, sinks, **more: seen.append((window, sinks)))
    c = host(blocks=40, max_context=160)
    q = torch.zeros(1, 1, 8, dtype=torch.float16)
    c.step([0], [100])
    c.step([1], [30])
    assert c.trim(0, window=10, sinks=5) == 20         # blocks 2 to 21: tokens 8 to 87
    both = c.step([0, 1], [1, 1])                      # (the token at 100 sees from 88 on under a window of 13)
    for window, sinks in ((0, 0), (14, 5), (10, 9), (0, 5)):
        with pytest.raises(ValueError, match="at most 13 tokens and 8 sinks"):
            c.attend(0, q, both, window=window, sinks=sinks)
    assert not seen
    for mask in ((13, 8), (10, 5), (1, 0)):
        c.attend(0, q, both, window=mask[0], sinks=mask[1])
    # requests with all of their blocks, or without tokens in the step, ask for nothing
    c.attend(0, q, c.step([1], [1]))
    c.attend(0, q, c.step([0, 1], [0, 1]))
    assert seen == [(13, 8), (10, 5), (1, 0), (0, 0), (0, 0)]
    c.free(0)
    c.attend(0, q, c.step([0], [1]))


@pytest.mark.parametrize("requests", [[0, 1, 2], [2, 0], [0]])
def test_a_step_keeps_its_tables(host, requests):
    c = host(blocks=40, max_context=160)
    c.step(requests, [30 + r for r in requests])
    s = c.step(requests, [2] * len(requests))
    before = s.tables.clone()
    assert c.trim(0, window=4) > 0
    assert torch.equal(s.tables, before)
    c.free(requests[-1])
    c.free(0)
    c.step([0], [9])
    assert torch.equal(s.tables, before)
    # and the cache's own go on
    s = c.step([0, 1, 2], [5, 5, 5])
    assert s.tables[0, :4].tolist() == c.tables[0, :4].tolist() and -1 not in s.tables[0, :4].tolist()
    used = [e for e in c.tables.flatten().tolist() if e >= 0]
    assert sorted(used + c._free.tolist()) == list(range(40))


def test_a_step_keeps_its_prefix(host):
    c = host()
    c.step([0], [6])
    c.share(0, 1)
    s = c.step([1], [2])
    before = s.prefix[0].clone(), s.tables.clone()
    c.free(1)
    c.free(0)
    c.step([0], [20])
    assert torch.equal(s.prefix[0], before[0]) and torch.equal(s.tables, before[1])


@pytest.mark.gpu
def test_a_trim_between_two_layers():
    c = cache(layers=2, dim=64, blocks=60, max_context=100, max_requests=1)
    gen = torch.Generator().manual_seed(5)
    draw = lambda *shape: torch.randn(*shape, 1, 64, generator=gen).half().cuda()
    q = draw(40)
    s = c.step([0], [80])
    k, v = draw(2, 80)
    for layer in (0, 1):
        c.write(layer, k, v, s)
    s = c.step([0], [20])
    k, v = draw(2, 20)
    c.write(0, k, v, s), c.write(1, k, v, s)
    out = [c.attend(0, q[:20], s, window=16)]
    assert c.trim(0, window=16) > 0
    out.append(c.attend(1, q[:20], s, window=16))
    assert torch.equal(out[0], out[1])


def test_requests_that_do_not_exist(host):
    """(A negative number would name a request by a second name, twice in one step.)"""
    c = host()
    c.step([2], [3])
    for call in (lambda: c.step([-1, 2], [1, 1]), lambda: c.step([3], [1]), lambda: c.free(-1), lambda: c.trim(-1, 4), lambda: c.share(-1, 0),
                 lambda: c.share(2, -3), lambda: c.length(-1)):
        with pytest.raises(IndexError, match="0 to 2"):
            call()
    assert c.length(2) == 3 and c.free_blocks == 11
