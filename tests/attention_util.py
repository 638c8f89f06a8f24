"""A paged cache filled from contiguous keys and values, and the attention over it in 64 bits."""
import math

import torch

# half a unit in the last place, relative
ROUNDING = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


class Step:
    """``requests``: (context, new tokens) each.  Blocks are dealt out at random; what no token may read is NaN: slots past a
    context, blocks of nobody, blocks behind a window (their table entries are -1 or point outside of the cache)."""

    def __init__(self, seed, requests, heads, kv_heads, dim, block_size, dtype=torch.float16, layout="token", window=0, sinks=0,
                 prefix=0, device="cuda", stale=-1, q_scale=2.0):
        gen = torch.Generator().manual_seed(seed)
        self.requests, self.window, self.sinks, self.prefix, self.dim = requests, window, sinks, prefix, dim
        self.heads, self.kv_heads, self.block_size, self.dtype = heads, kv_heads, block_size, dtype
        rand = lambda *shape: torch.randn(*shape, generator=gen).to(dtype).to(device)
        own = [-(-c // block_size) for c, _ in requests]
        shared = -(-prefix // block_size)
        blocks = sum(own) + shared + 2
        order = torch.randperm(blocks, generator=gen)
        shape = (2, blocks, block_size, kv_heads, dim) if layout == "token" else (2, blocks, kv_heads, block_size, dim)
        cache = torch.full(shape, float("nan"), dtype=dtype, device=device)
        if layout == "head":
            cache = cache.transpose(2, 3)
        self.k_cache, self.v_cache = cache[0], cache[1]
        width = max(own, default=0) + 2
        tables = torch.full((len(requests), width), stale, dtype=torch.int32)
        self.k, self.v = [], []           # per request [prefix + context, kv_heads, dim]
        pk, pv = rand(prefix, kv_heads, dim), rand(prefix, kv_heads, dim)
        self.prefix_blocks = order[:shared].to(torch.int32).to(device)
        self._fill(order[:shared], pk, pv, 0)
        at = shared
        for b, (c, n) in enumerate(requests):
            k, v = rand(c, kv_heads, dim), rand(c, kv_heads, dim)
            self.k.append(torch.cat([pk, k]))
            self.v.append(torch.cat([pv, v]))
            lo = max(0, c - n + 1 - window) if window else 0
            mine = order[at:at + own[b]]
            seen = [j for j in range(own[b]) if (j + 1) * block_size > lo or j * block_size < min(sinks, lo)]
            tables[b, seen] = mine[seen].to(torch.int32)
            for j in seen:
                self._fill(mine[j:j + 1], k[j * block_size:], v[j * block_size:], 0)
            at += own[b]
        self.tables = tables.to(device)
        counts = torch.tensor([n for _, n in requests], dtype=torch.int32)
        self.starts = torch.cat([torch.zeros(1, dtype=torch.int32), counts.cumsum(0, dtype=torch.int32)]).to(device)
        self.contexts = torch.tensor([c for c, _ in requests], dtype=torch.int32, device=device)
        self.tokens = int(counts.sum())
        self.q = rand(self.tokens, heads, dim).mul_(q_scale)
        self.most = max((c for c, _ in requests), default=0)

    def _fill(self, blocks, k, v, start):
        for i, b in enumerate(blocks.tolist()):
            part = slice(start + i * self.block_size, start + (i + 1) * self.block_size)
            n = len(k[part])
            self.k_cache[b, :n], self.v_cache[b, :n] = k[part], v[part]

    def expected(self, scale=None):
        """(attention in 64 bits, the same with |v| in place of v) [tokens, heads, dim]."""
        scale = scale or 1 / math.sqrt(self.dim)
        out = torch.zeros(self.tokens, self.heads, self.dim, dtype=torch.float64, device=self.q.device)
        size = torch.zeros_like(out)
        begin, group = 0, self.heads // self.kv_heads
        for b, (c, n) in enumerate(self.requests):
            k, v = self.k[b].double(), self.v[b].double()
            p = torch.arange(c - n, c, device=out.device)[:, None]
            j = torch.arange(-self.prefix, c, device=out.device)[None]
            sees = (j < 0) | (j <= p)
            if self.window:
                sees &= (j > p - self.window) | (j < self.sinks)
            for h in range(self.heads):
                g = h // group
                s = (self.q[begin:begin + n, h].double() @ k[:, g].T * scale).masked_fill(~sees, -math.inf)
                w = torch.softmax(s, 1) if s.shape[1] else s
                w = torch.where(sees.any(1, keepdim=True), w, 0.0)
                out[begin:begin + n, h] = w @ v[:, g]
                size[begin:begin + n, h] = w @ v[:, g].abs()
            begin += n
        return out, size


def assert_attention(got, step, what, scale=None):
    """Two roundings to the cache's type, of the softmax's shares and of the result: 2 u of the sum of |share * value|, and a
    quarter of u for what 32-bit scores add (their relative error is at most some tens of 2^-24, times |score| below 16,
    below u / 4 for fp16), and the smallest fp16 steps."""
    want, size = step.expected(scale)
    assert got.shape == want.shape and got.dtype == step.dtype, (what, got.shape, got.dtype)
    err = (got.double() - want).abs()
    bound = 2.25 * ROUNDING[step.dtype] * size + 2.0 ** -24
    bad = ~(err <= bound)
    assert not bool(bad.any()), (f"{what}: {int(bad.sum())} of {bad.numel()} out of bounds, the first at "
                                 f"{[int(x) for x in bad.nonzero()[0]]}, worst {float((err / bound).nan_to_num(1e9).max()):.3g} bounds")
