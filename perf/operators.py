"""The performance cases of the operators around the quantised layers in a serving step: a paged key/value cache and the
attention that reads it.

A case is one call of one of four operators:

* ``tables``: block tables, slot maps, query offsets and positions of a step, from the lengths of the requests;
* ``write``: the step's keys and values into the slots of the cache;
* ``attend``: the attention of the step's tokens over their requests' blocks, causal, with or without a sliding window and
  first tokens that stay visible (sinks);
* ``prefix``: the same for a batch whose requests share a long prefix, which is read once for all of them.

``requests`` requests take part in a step.  The longest has ``context`` tokens when the step is done, ``tokens`` of them new;
``spread`` says how the others lie below that: all alike ("even") or over the logarithm ("log").  ``block`` is the number of
tokens in a block of the cache.  ``layout`` names the order of a cache in memory: "token" [blocks, block, heads, dim] or "head"
[blocks, heads, block, dim]; ``fused`` says that q, k and v are columns of one product's output, as
``fuse_shared_input_layers`` leaves them.
"""
import math

import torch

own = False

FLOPS = 4 * 128 * 32 * 8192 * 8193 // 2     # the largest listed attention; drawn ones stay within both figures
BYTES = 2 * 2 * 16 * 32768 * 8 * 128
SCORES = 32 * 8192 * 8192                   # scores that the plain form holds at once


def _case(name, op, **more):
    case = {"name": name, "op": op, "dtype": "float16", "heads": 32, "kv_heads": 8, "dim": 128, "block": 16, "requests": 1,
            "context": 1, "tokens": 1, "spread": "even", "window": 0, "sinks": 0, "prefix": 0, "layout": "token",
            "fused": False}
    case.update(more)
    return case


def listed():
    return [
        # the bookkeeping of a decoding step of a batch, and of a step that takes in prompts of very different lengths
        _case("tables-decode-64", "tables", requests=64, context=4096, spread="log"),
        _case("tables-prompts-333", "tables", requests=333, context=9000, tokens=4099, spread="log"),
        # keys and values of a decoding step of a batch, and of a long prompt out of a fused q/k/v product
        _case("write-decode-64", "write", requests=64, context=1024, spread="log"),
        _case("write-prompt-8192", "write", dtype="bfloat16", context=8192, tokens=8192, fused=True),
        # decoding: one short conversation, where latency counts; a batch of long ones under a window with sinks, whose
        # blocks behind the window were given back; a batch of long documents, the call that is bound by memory
        _case("decode-1x512", "attend", context=512),
        _case("decode-64-window4096", "attend", requests=64, context=32768, spread="log", window=4096, sinks=4, block=64),
        _case("decode-16x32768", "attend", requests=16, context=32768, layout="head", block=64),
        # prompts: under a window with sinks, in bfloat16 out of a fused product; a long one without; pieces of prompts of
        # ragged lengths behind contexts that are in the cache, narrow heads in sevens, blocks that are no power of two
        _case("prompt-4096-window1024", "attend", dtype="bfloat16", context=4096, tokens=4096, window=1024, sinks=4,
              fused=True),
        _case("prompt-8192", "attend", context=8192, tokens=8192, block=64),
        _case("chunks-5x333-dim80", "attend", dtype="bfloat16", heads=28, kv_heads=4, dim=80, block=24, requests=5,
              context=9001, tokens=333, spread="log"),
        # a small batch behind one instruction prompt, and many questions to one long document
        _case("prefix-decode-8x1000", "prefix", requests=8, context=37, prefix=1000, spread="log"),
        _case("prefix-decode-128x16384", "prefix", dtype="bfloat16", requests=128, context=512, prefix=16384, spread="log",
              block=64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("tables", "write", "attend", "attend", "attend", "attend", "prefix", "prefix"))
    kv_heads = rng.choice((1, 2, 4, 8, 8, 8, 16, 32))
    group = rng.choice([g for g in (1, 1, 4, 4, 5, 7, 8, 16) if g * kv_heads <= 64])
    c = {"op": op, "dtype": rng.choice(("float16", "float16", "bfloat16")), "heads": group * kv_heads, "kv_heads": kv_heads,
         "dim": rng.choice((64, 128, 128, 128, 80, 96, 256)), "block": rng.choice((16, 16, 32, 64, 128, 24, 7)),
         "requests": _log(rng, 1, 256), "context": _log(rng, 16, 32768), "tokens": 1, "spread": rng.choice(("even", "log", "log")),
         "window": 0, "sinks": 0, "prefix": 0, "layout": rng.choice(("token", "head")), "fused": rng.random() < 0.3}
    if op in ("tables", "write") and rng.random() < 0.6 or op == "attend" and rng.random() < 0.5:
        c["tokens"] = _log(rng, 1, min(c["context"], 8192))     # prompts, or pieces of them
    if op == "attend" and rng.random() < 0.5:
        c["window"], c["sinks"] = _log(rng, 64, 8192), rng.choice((0, 1, 4, 33))
    if op == "prefix":
        c["prefix"], c["context"] = _log(rng, 128, 32768), _log(rng, 1, 4096)
        if rng.random() < 0.3:
            c["tokens"] = _log(rng, 1, min(c["context"], 16))

    def fits():
        w, b = work(c), c["requests"]
        seen = _width(c) + c["prefix"]
        return (w["flops"] <= FLOPS and w["bytes"] <= BYTES and b * c["heads"] * c["tokens"] * seen <= SCORES
                and b * seen * c["kv_heads"] * c["dim"] * 4 <= BYTES)
    while not fits():
        k = rng.choice([k for k in ("requests", "context", "tokens", "prefix") if c[k] > 1])
        c[k] = c[k] * 3 // 4
        c["tokens"] = min(c["tokens"], c["context"])
    return c


# ------------------------------------------------------------------ lengths, which follow from the case alone
def _part(most, i, ratio, spread):
    return most if spread == "even" else max(1, round(most ** (1.0 - i * ratio % 1.0)))


def _lengths(case):
    """(context, new tokens) of every request: the first has the largest, the others follow two irrational steps."""
    new = [_part(case["tokens"], i, 0.7548776662, case["spread"]) for i in range(case["requests"])]
    return [(max(n, _part(case["context"], i, 0.6180339887, case["spread"])), n) for i, n in enumerate(new)]


def _seen(case, context, n):
    """(first tokens that are seen for being sinks, first token of the window) of a request's new tokens together."""
    lo = max(0, context - n + 1 - case["window"]) if case["window"] else 0
    return min(case["sinks"], lo), lo


def _width(case):
    return max(s + c - lo for c, n in _lengths(case) for s, lo in [_seen(case, c, n)])


def _pairs(case, context, n):
    """Pairs of a new token and a token of its context that it sees."""
    def capped(x, most):    # 1 + 2 + ... + x, each term at most `most`
        x = max(0, x)
        low = min(x, most)
        return low * (low + 1) // 2 + (x - low) * most
    if not case["window"]:
        return capped(context, context) - capped(context - n, context)
    w, s = case["window"], case["sinks"]
    return capped(context, w) - capped(context - n, w) + capped(context - w, s) - capped(context - n - w, s)


def work(case):
    lengths = _lengths(case)
    T = sum(n for _, n in lengths)
    D, hq, hk, blk = case["dim"], case["heads"], case["kv_heads"], case["block"]
    if case["op"] == "tables":
        new = sum(-(-c // blk) - -(-(c - n) // blk) for c, n in lengths)
        return {"bytes": 4 * (2 * len(lengths) + 2 * new + 2 * T + 2 * len(lengths) + 2), "flops": T}
    if case["op"] == "write":
        return {"bytes": 2 * 2 * 2 * T * hk * D + 4 * T, "flops": 0}
    rows = sum(s + c - lo for c, n in lengths for s, lo in [_seen(case, c, n)]) + case["prefix"]
    pairs = sum(_pairs(case, c, n) for c, n in lengths) + T * case["prefix"]
    return {"bytes": 2 * 2 * rows * hk * D + 2 * 2 * T * hq * D + 4 * (rows // blk + 2 * len(lengths)),
            "flops": 4 * pairs * hq * D}


# ------------------------------------------------------------------ inputs
def _cache(case, blocks, dtype, gen):
    b, h, d = case["block"], case["kv_heads"], case["dim"]
    if case["layout"] == "token":
        both = torch.randn((2, blocks, b, h, d), device="cuda", generator=gen, dtype=dtype)
    else:
        both = torch.randn((2, blocks, h, b, d), device="cuda", generator=gen, dtype=dtype).transpose(2, 3)
    return both[0], both[1]


def _new(case, T, dtype, gen):
    """q, k and v of a step's tokens."""
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if case["fused"]:
        qkv = torch.randn((T, (hq + 2 * hk) * d), device="cuda", generator=gen, dtype=dtype)
        q, k, v = qkv.split((hq * d, hk * d, hk * d), dim=1)
        return q.view(T, hq, d).mul_(2), k.view(T, hk, d), v.view(T, hk, d)
    q = torch.randn((T, hq, d), device="cuda", generator=gen, dtype=dtype).mul_(2)
    return q, *(torch.randn((T, hk, d), device="cuda", generator=gen, dtype=dtype) for _ in range(2))


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, blk = getattr(torch, case["dtype"]), case["block"]
    lengths = _lengths(case)
    T = sum(n for _, n in lengths)
    most = max(c for c, _ in lengths)
    wide = -(-most // blk) + 3                                   # the tables have room for what comes
    state = {"case": case, "T": T, "most": most, "seen": _width(case), "tokens": max(n for _, n in lengths)}
    if case["op"] == "tables":
        held = [-(-(c - n) // blk) for c, n in lengths]
        new = sum(-(-c // blk) for c, _ in lengths) - sum(held)
        ids = torch.randperm(sum(held) + new + 64, device="cuda", generator=gen).to(torch.int32)
        tables = torch.full((len(lengths), wide), -1, dtype=torch.int32, device="cuda")
        at = 0
        for b, h in enumerate(held):
            tables[b, :h] = ids[at:at + h]
            at += h
        state.update(lengths=_ints([c - n for c, n in lengths]), counts=_ints([n for _, n in lengths]), tables=tables,
                     free=ids[at:].clone())
        return state
    if case["op"] == "write":
        blocks = sum(-(-c // blk) for c, _ in lengths) + 3
        order = torch.randperm(blocks, device="cuda", generator=gen)
        slots, at = [], 0
        for c, n in lengths:
            p = torch.arange(c - n, c, device="cuda")
            slots.append(order[at + p // blk] * blk + p % blk)
            at += -(-c // blk)
        _, k, v = _new(case, T, dtype, gen)
        k_cache, v_cache = _cache(case, blocks, dtype, gen)
        state.update(k=k, v=v, k_cache=k_cache, v_cache=v_cache, slots=torch.cat(slots).to(torch.int32))
        return state
    # blocks that no new token sees, behind a window, were given back: the tables hold -1 there
    kept = [[j for j in range(-(-c // blk)) if j * blk < s or (j + 1) * blk > lo] for c, n in lengths for s, lo in [_seen(case, c, n)]]
    shared = -(-case["prefix"] // blk)
    blocks = sum(map(len, kept)) + shared + 3
    order = torch.randperm(blocks, device="cuda", generator=gen).to(torch.int32)
    k_cache, v_cache = _cache(case, blocks, dtype, gen)
    tables = torch.full((len(lengths), wide), -1, dtype=torch.int32, device="cuda")
    at = shared
    for b, own_blocks in enumerate(kept):
        tables[b, torch.tensor(own_blocks, device="cuda")] = order[at:at + len(own_blocks)]
        at += len(own_blocks)
    # slots that nobody has written yet hold whatever was there
    ends = [(int(order[shared - 1]) if shared else 0, case["prefix"] % blk if shared else 0)]
    last = torch.cumsum(torch.tensor([len(x) for x in kept]), 0) + shared - 1
    ends += list(zip(order.cpu()[last].tolist(), [c % blk for c, _ in lengths]))
    for block, used in ends:
        if used:
            k_cache[block, used:] = float("nan")
            v_cache[block, used:] = float("nan")
    starts = [0]
    for _, n in lengths:
        starts.append(starts[-1] + n)
    q, _, _ = _new(case, T, dtype, gen)
    state.update(q=q, k_cache=k_cache, v_cache=v_cache, tables=tables, starts=_ints(starts),
                 contexts=_ints([c for c, _ in lengths]), shared=order[:shared].clone())
    return state


# ------------------------------------------------------------------ the framework's calls
def _own(state):
    from autogptq.tvm_amd import attention

    c, s = state["case"], state
    if c["op"] == "tables":
        made = attention.cache_tables(s["lengths"], s["counts"], s["tables"], s["free"], s["T"], c["block"])
        return [s["tables"], *made]
    if c["op"] == "write":
        attention.cache_write(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"])
        return [s["k_cache"], s["v_cache"]]
    if c["op"] == "attend":
        return attention.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["starts"], s["contexts"],
                                         max_context=s["most"], window=c["window"], sinks=c["sinks"])
    return attention.shared_prefix_attention(s["q"], s["k_cache"], s["v_cache"], s["shared"], c["prefix"], s["tables"],
                                             s["starts"], s["contexts"], max_context=s["most"])


# ------------------------------------------------------------------ the plain forms
def _before(x):
    """Sums of what stands before each entry, and the whole sum behind the last."""
    return torch.nn.functional.pad(torch.cumsum(x, 0, dtype=torch.int32), (1, 0))


def _owner(starts, T):
    return torch.searchsorted(starts[1:].contiguous(), torch.arange(T, dtype=torch.int32, device=starts.device), right=True)


def _plain_tables(s):
    blk, T, tables, free = s["case"]["block"], s["T"], s["tables"], s["free"]
    starts, contexts = _before(s["counts"]), s["lengths"] + s["counts"]
    held, need = (s["lengths"] + blk - 1) // blk, (contexts + blk - 1) // blk
    before = _before(need - held)
    j = torch.arange(tables.shape[1], dtype=torch.int32, device=tables.device)[None]
    from_free = free[(before[:-1, None] + j - held[:, None]).clamp(0, free.numel() - 1)]
    tables.copy_(torch.where((j >= held[:, None]) & (j < need[:, None]), from_free, tables))
    who = _owner(starts, T)
    positions = s["lengths"][who] + torch.arange(T, dtype=torch.int32, device=tables.device) - starts[who]
    slots = tables[who, positions // blk] * blk + positions % blk
    return [tables, starts, contexts, slots, positions, before[-1:]]


def _plain_write(s):
    blk = s["case"]["block"]
    block, at = s["slots"] // blk, s["slots"] % blk
    s["k_cache"][block, at] = s["k"]
    s["v_cache"][block, at] = s["v"]
    return [s["k_cache"], s["v_cache"]]


def _rows(cache, tables, at, there):
    """The cache's rows at the positions `at` of every request, [requests, heads, positions, dim] in 32 bits; zeros where
    there is none."""
    blk = cache.shape[1]
    block = torch.gather(tables, 1, torch.where(there, at // blk, 0).long())
    rows = cache[torch.where(there, block, 0), torch.where(there, at % blk, 0)].float()
    return torch.where(there[:, :, None, None], rows, 0.0).transpose(1, 2)


def _plain_attend(s):
    c, q, dev = s["case"], s["q"], s["q"].device
    T, hq, D = q.shape
    hk, w, sinks = c["kv_heads"], c["window"], c["sinks"]
    starts, contexts = s["starts"], s["contexts"]
    counts = starts[1:] - starts[:-1]
    B, N, V = contexts.shape[0], s["tokens"], s["seen"]
    lo = (contexts - counts + 1 - w).clamp_min(0) if w else torch.zeros_like(contexts)
    first = lo.clamp_max(sinks)[:, None]
    i = torch.arange(V, dtype=torch.int32, device=dev)[None]
    at = torch.where(i < first, i, i - first + lo[:, None])                         # [B, V]
    there = at < contexts[:, None]
    keys, values = (_rows(s[n], s["tables"], at, there) for n in ("k_cache", "v_cache"))
    t = torch.arange(N, dtype=torch.int32, device=dev)[None]
    row = q[(starts[:-1, None] + t).clamp_max(T - 1)].float()                       # [B, N, hq, D]
    row = row.view(B, N, hk, hq // hk, D).permute(0, 2, 3, 1, 4).reshape(B, hk, -1, D)
    p = ((contexts - counts)[:, None] + t)[:, :, None]                              # [B, N, 1]
    at, there = at[:, None], there[:, None]
    sees = there & (at <= p)
    if w:
        sees &= (at > p - w) | (at < sinks)
    scores = (row @ keys.transpose(2, 3).contiguous()).mul_(1 / math.sqrt(D))
    scores = scores.view(B, hk, hq // hk, N, V).masked_fill_(~sees[:, None, None], float("-inf")).view(B, hk, -1, V)
    if c["prefix"]:
        j = torch.arange(c["prefix"], device=dev)[None]
        all_there = torch.ones_like(j, dtype=torch.bool)
        keys0, values0 = (_rows(s[n], s["shared"][None], j, all_there)[0] for n in ("k_cache", "v_cache"))
        scores0 = (row @ keys0.transpose(1, 2).contiguous()).mul_(1 / math.sqrt(D))
        top = torch.maximum(scores.amax(-1, keepdim=True), scores0.amax(-1, keepdim=True))
        scores0 = scores0.sub_(top).exp_()
    else:
        top = scores.amax(-1, keepdim=True)
        top = torch.where(torch.isinf(top), 0.0, top)
    scores = scores.sub_(top).exp_()
    total = scores.sum(-1, keepdim=True)
    out = scores @ values
    if c["prefix"]:
        total = total + scores0.sum(-1, keepdim=True)
        out = out + scores0 @ values0
    out = torch.where(total > 0, out / total, 0.0)
    out = out.view(B, hk, hq // hk, N, D).permute(0, 3, 1, 2, 4).reshape(B, N, hq, D)
    who = _owner(starts, T)
    return out[who, torch.arange(T, device=dev) - starts[who]].to(q.dtype)


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    return _plain_tables(state) if op == "tables" else _plain_write(state) if op == "write" else _plain_attend(state)


# ------------------------------------------------------------------ the definition, in 64 bits
def exact(case, seed):
    s, blk, lengths = prepare(case, seed), case["block"], _lengths(case)
    if case["op"] == "tables":
        tables, free = s["tables"].cpu().tolist(), s["free"].cpu().tolist()
        starts, slots, positions, taken = [0], [], [], 0
        for b, (c, n) in enumerate(lengths):
            for p in range(c - n, c):
                if p % blk == 0:
                    tables[b][p // blk] = free[taken]
                    taken += 1
                positions.append(p)
                slots.append(tables[b][p // blk] * blk + p % blk)
            starts.append(starts[-1] + n)
        return [_ints(x) for x in (tables, starts, [c for c, _ in lengths], slots, positions, [taken])]
    if case["op"] == "write":
        if s["T"] > 100000:
            return None
        out = []
        for name in ("k", "v"):
            cache = s[name + "_cache"].double()
            for i, slot in enumerate(s["slots"].tolist()):
                cache[slot // blk, slot % blk] = s[name][i].double()
            out.append(cache)
        return out
    T, hq, D = s["q"].shape
    hk, w = case["kv_heads"], case["window"]
    out = torch.zeros((T, hq, D), dtype=torch.float64, device="cuda")
    k0, v0 = (x[s["shared"]].flatten(0, 1)[:case["prefix"]].double() for x in (s["k_cache"], s["v_cache"]))
    begin = 0
    for b, (c, n) in enumerate(lengths):
        seen_first, lo = _seen(case, c, n)
        at = torch.cat([torch.arange(seen_first, device="cuda"), torch.arange(lo, c, device="cuda")])
        block = s["tables"][b].long()[at // blk]
        k = torch.cat([k0, s["k_cache"][block, at % blk].double()])
        v = torch.cat([v0, s["v_cache"][block, at % blk].double()])
        step = max(1, 2 ** 27 // k.shape[0])
        for t in range(0, n, step):
            m = min(step, n - t)
            p = torch.arange(c - n + t, c - n + t + m, device="cuda")[:, None]
            hidden = at > p
            if w:
                hidden |= (at <= p - w) & (at >= case["sinks"])
            hidden = torch.cat([torch.zeros((m, k0.shape[0]), dtype=torch.bool, device="cuda"), hidden], 1)
            for h in range(hq):
                g = h // (hq // hk)
                logits = s["q"][begin + t:begin + t + m, h].double() @ k[:, g].T / D ** 0.5
                out[begin + t:begin + t + m, h] = torch.softmax(logits.masked_fill(hidden, -math.inf), 1) @ v[:, g]
        begin += n
    return out
