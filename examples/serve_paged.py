"""A small GPTQ decoder served from a paged cache: a shared instruction prompt, a batch of requests behind it, decoding, and a
long conversation under a sliding window.

    python examples/serve_paged.py

Random weights of random layers (there is no checkpoint here), the quantised layers of this package for every product, and
``PagedCache`` with the attention that reads it between them.  Every step's logits are compared with a plain evaluation of the
same model over the whole sequences.  Then the same from a cache in 4 bits, where every layer's attention is compared with a plain one
over the keys and values that the cache gives back.  (Not the logits: a value that two evaluations put a hair apart may be rounded to
different codes, and layers upon layers of a random model make much of it.)"""
import math
import os
import sys

import torch
import torch.nn as nn

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from autogptq.tvm_amd import PagedCache, QuantLinear, fuse_shared_input_layers  # noqa: E402
from autogptq.tvm_amd.pack import synth_layer  # noqa: E402

HIDDEN, HEADS, KV_HEADS, DIM, INNER, VOCAB, LAYERS = 512, 8, 2, 64, 1024, 256, 2


def _quantised(seed, k, n):
    w = synth_layer(seed, k, n, 4, 128, False)
    layer = QuantLinear(4, 128, k, n, False)
    layer.load_state_dict({name: w[name] for name in ("qweight", "qzeros", "scales", "g_idx")})
    return layer


def _normed(x):
    return (x.float() * torch.rsqrt(x.float().pow(2).mean(-1, keepdim=True) + 1e-5)).half()


def _rotated(x, positions):
    """Rotary embedding of [tokens, heads, dim]."""
    half = x.shape[-1] // 2
    angle = positions[:, None].float() * torch.exp(torch.arange(half, device=x.device) * (-math.log(10000.0) / half))
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    a, b = x.float().chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).half()


class Block(nn.Module):
    def __init__(self, seed):
        super().__init__()
        shapes = {"q_proj": (HIDDEN, HEADS * DIM), "k_proj": (HIDDEN, KV_HEADS * DIM), "v_proj": (HIDDEN, KV_HEADS * DIM),
                  "o_proj": (HEADS * DIM, HIDDEN), "gate_proj": (HIDDEN, INNER), "up_proj": (HIDDEN, INNER), "down_proj": (INNER, HIDDEN)}
        for i, (name, (k, n)) in enumerate(shapes.items()):
            setattr(self, name, _quantised(seed + i, k, n))

    def forward(self, h, positions, attend):
        x = _normed(h)
        q, k, v = self.q_proj(x), self.k_proj(x), self.v_proj(x)
        q, k = _rotated(q.view(-1, HEADS, DIM), positions), _rotated(k.view(-1, KV_HEADS, DIM), positions)
        a = attend(q, k, v.view(-1, KV_HEADS, DIM))
        h = h + _normed(self.o_proj(a.reshape(-1, HEADS * DIM)))
        x = _normed(h)
        return h + _normed(self.down_proj(_normed(torch.nn.functional.silu(self.gate_proj(x)) * self.up_proj(x))))


class Decoder(nn.Module):
    def __init__(self, seed=1):
        super().__init__()
        gen = torch.Generator().manual_seed(seed)
        self.register_buffer("embedding", torch.randn(VOCAB, HIDDEN, generator=gen).half())
        self.blocks = nn.ModuleList(Block(100 * seed + 10 * i) for i in range(LAYERS))

    def _run(self, tokens, positions, attend):
        h = self.embedding[tokens]
        for i, block in enumerate(self.blocks):
            h = block(h, positions, lambda q, k, v: attend(i, q, k, v))
        return _normed(h).float() @ self.embedding.float().t()

    @torch.no_grad()
    def step(self, cache, requests, tokens, window=0, sinks=0, watch=None):
        """Logits of the new tokens (one 1-D tensor a request), which are in the cache afterwards."""
        step = cache.step(requests, [t.numel() for t in tokens])

        def attend(layer, q, k, v):
            cache.write(layer, k, v, step)
            out = cache.attend(layer, q, step, window=window, sinks=sinks)
            if watch:
                watch(layer, q, out)
            return out
        return self._run(torch.cat(tokens), step.positions, attend)

    @torch.no_grad()
    def plain(self, tokens, window=0, sinks=0):
        """The same over one whole sequence, with the attention as torch operations in 32 bits."""
        p = torch.arange(tokens.numel(), device=tokens.device)
        return self._run(tokens, p, lambda layer, q, k, v: _attention(q, k, v, window, sinks))


def _attention(q, k, v, window=0, sinks=0):
    """Causal attention of the last len(q) of len(k) tokens."""
    j = torch.arange(len(k), device=q.device)
    p = j[len(k) - len(q):, None]
    sees = j[None] <= p
    if window:
        sees &= (j[None] > p - window) | (j[None] < sinks)
    k, v = (x.float().repeat_interleave(HEADS // KV_HEADS, 1).transpose(0, 1).contiguous() for x in (k, v))
    s = q.float().transpose(0, 1) @ k.transpose(1, 2).contiguous() / math.sqrt(DIM)
    return (torch.softmax(s.masked_fill(~sees, -math.inf), -1) @ v).transpose(0, 1).half()


def main(device="cuda:0", verbose=True, quantize=None):
    model = Decoder().to(device).eval()
    fuse_shared_input_layers(model)
    gen = torch.Generator().manual_seed(3)
    draw = lambda n: torch.randint(0, VOCAB, (n,), generator=gen).to(device)
    cache = PagedCache(LAYERS, blocks=96, block_size=16, kv_heads=KV_HEADS, dim=DIM, max_requests=6, max_context=640, device=device,
                       quantize=quantize)
    worst = 0.0

    def compare(got, want, what):
        nonlocal worst
        off = float((got.float() - want.float()).norm() / want.float().norm())
        worst = max(worst, off)
        assert off < 2e-2, f"{what}: {off}"
        if verbose:
            print(f"{what}: relative difference {off:.2g}", flush=True)

    def check(got, whole, what, **mask):
        if not quantize:
            compare(got, model.plain(whole, **mask)[-got.shape[0]:], what)

    def step(requests, tokens, **mask):
        def watch(layer, q, out):
            at = 0
            for r, n in zip(requests, map(len, tokens)):
                k, v = cache.read(layer, r)
                if r in behind:
                    k, v = (torch.cat([a[:behind[r]], b]) for a, b in zip(cache.read(layer, 0), (k, v)))
                compare(out[at:at + n], _attention(q[at:at + n], k, v, **mask), f"layer {layer} of request {r} at {len(k)} tokens")
                at += n
        return model.step(cache, requests, tokens, watch=watch if quantize else None, **mask)
    behind = {}         # tokens of request 0 that a request stands behind

    # an instruction prompt, then four requests behind it with prompts of their own, then decoding together
    instructions = draw(100)
    check(step([0], [instructions]), instructions, "instructions of 100 tokens")
    requests = [1, 2, 3, 4]
    for r in requests:
        cache.share(0, r)
        behind[r] = instructions.numel()
    texts = [draw(n) for n in (7, 33, 1, 64)]
    logits = step(requests, texts)
    ends = torch.tensor([t.numel() for t in texts]).cumsum(0) - 1
    for n in range(8):
        for i, r in enumerate(requests):
            rows = logits[ends[i]:ends[i] + 1]
            check(rows, torch.cat([instructions, texts[i]]), f"request {r} at {100 + texts[i].numel()} tokens")
        new = [logits[e].argmax()[None] for e in ends]
        texts = [torch.cat([t, x]) for t, x in zip(texts, new)]
        logits, ends = step(requests, new), torch.arange(4)
    for r in requests:
        cache.free(r)

    # a long conversation under a window of 48 tokens and 4 sinks, its old blocks given back as it goes
    text, mask = draw(200), dict(window=48, sinks=4)
    check(step([5], [text], **mask), text, "conversation of 200 tokens under a window", **mask)
    for n in range(24):
        cache.trim(5, **mask)
        new = draw(1 + n % 3)
        text = torch.cat([text, new])
        check(step([5], [new], **mask), text, f"conversation of {text.numel()} tokens", **mask)
    cache.free(5)
    cache.free(0)
    assert cache.free_blocks == 96
    return worst


if __name__ == "__main__":
    print(f"done, largest relative difference {main():.2g}")
    print(f"from a cache in 4 bits, largest relative difference of an attention {main(quantize='mxfp4'):.2g}")
