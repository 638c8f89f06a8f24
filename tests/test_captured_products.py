"""Products of quantised layers in captured graphs, beside eager calls and captures that come later."""
import pytest
import torch

from autogptq.tvm_amd import QuantLinear
from autogptq.tvm_amd.pack import synth_layer

pytestmark = pytest.mark.gpu


def make(seed, K, N, bits=4):
    w = synth_layer(seed, K, N, bits, 128, True)
    q = QuantLinear(bits, 128, K, N, True)
    q.load_state_dict({k: w[k] for k in ("qweight", "qzeros", "scales", "g_idx")}, strict=False)
    return q.cuda()


def overwrite():
    """Fills what the allocator can hand out, on the current stream, with bytes that are no zeros."""
    return [torch.full((1 << k,), 0x7f, dtype=torch.uint8, device="cuda") for k in range(9, 28)] + [
        torch.full((16 << 20,), 0x7f, dtype=torch.uint8, device="cuda") for _ in range(16)]


def capture(stream, call):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = call()
    return graph, got


# 11008 columns: the decode kernel's halved tiles meet in the slots of a workspace that is zero between launches
@pytest.mark.parametrize("K, N", [(1024, 11008), (4096, 1024)])
def test_replays_after_calls_that_need_more(K, N):
    q = make(7, K, N)
    gen = torch.Generator().manual_seed(8)
    xs = {M: torch.randn(M, K, generator=gen).half().cuda() for M in (1, 3, 24, 60, 300, 2000)}
    want = {M: q(x) for M, x in xs.items()}
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    for M in (1, 3, 24, 60):
        graph, got = capture(stream, lambda: q(xs[M]))
        for _ in range(3):
            with torch.cuda.stream(stream):
                later = {n: q(x) for n, x in xs.items()}
                junk = overwrite()
                got.zero_()
                graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want[M]), M
            assert all(torch.equal(y, want[n]) for n, y in later.items())
            assert all(bool((j == 0x7f).all()) for j in junk), "a replay wrote into another tensor"
            del junk


def test_captures_replay_in_any_order():
    layers = [make(9, 1024, 11008), make(10, 1024, 11008, 3), make(11, 4096, 1024)]
    gen = torch.Generator().manual_seed(12)
    xs = [torch.randn(M, q.infeatures, generator=gen).half().cuda() for q, M in zip(layers, (1, 2, 40))]
    want = [q(x) for q, x in zip(layers, xs)]
    junk = overwrite()
    torch.cuda.synchronize()
    del junk
    torch.cuda.empty_cache()
    stream = torch.cuda.Stream()
    made = [capture(stream, lambda q=q, x=x: q(x)) for q, x in zip(layers, xs)]
    for order in ((1, 0, 2), (2, 1, 0), (0, 0, 1), (1, 2, 2)):
        for i in order:
            made[i][1].zero_()
            made[i][0].replay()
        torch.cuda.synchronize()
        for i in set(order):
            assert torch.equal(made[i][1], want[i]), (order, i)


def test_gradients_replay_after_calls_that_need_more():
    """(The gradient's calls go through the front end in Python, which keeps workspaces of its own.)"""
    K, N = 2176, 4096
    q = make(13, K, N)
    gen = torch.Generator().manual_seed(14)
    gs = {M: torch.randn(M, N, generator=gen).half().cuda() for M in (20, 38, 70, 300, 1000)}
    want = {M: q.grad_input(g) for M, g in gs.items()}
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    made = {M: capture(stream, lambda: q.grad_input(gs[M])) for M in (20, 38, 70)}
    for order in ((38, 20, 70), (70, 38), (20, 70)):
        with torch.cuda.stream(stream):
            later = {n: q.grad_input(g) for n, g in gs.items()}
            junk = overwrite()
            for M in order:
                made[M][1].zero_()
                made[M][0].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(made[M][1], want[M]) for M in order), order
        assert all(torch.equal(y, want[n]) for n, y in later.items())
        assert all(bool((j == 0x7f).all()) for j in junk), "a replay wrote into another tensor"
        del junk
