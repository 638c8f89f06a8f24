"""The performance cases of a paged key/value cache held in 4 bits: the write that quantises a step's keys and values, the read
that gives them back, and the attention that reads such a cache.

The format is MXFP4.  A head's ``dim`` values of a token are padded with zeros to a multiple of 32 and cut into groups of 32.  A
group has a power of two 2^e, kept as the byte e + 127, and 32 codes of 4 bits: a sign and one of 0, 1/2, 1, 3/2, 2, 3, 4, 6.  Byte
j of a row holds the values 2 j (low half) and 2 j + 1; a row has ``dim`` / 32, rounded up, groups of 16 bytes, and its scales
lie in 2 bytes (dim up to 64), 4 (up to 128) or 8.  With 2^x the power of two at or below the largest magnitude m of a group, e is
x - 2, or x - 1 where m >= 1.75 2^x (which would round up to the next power), kept within -23 .. 13 (float16) or -125 .. 125
(bfloat16).  Codes are the nearest ones, ties to the even code, and values beyond 6 2^e become that.  A group that holds an
infinity or a NaN has the scale byte 255 and stands for NaN.

A case is one call of one of four operators (the first: two calls):

* ``store``: a step's keys and values into the slots of the cache, and read back from them;
* ``read``: the keys and values of a whole request;
* ``attend``: the attention of the step's tokens over their requests' blocks, causal, with or without a sliding window and
  first tokens that stay visible (sinks);
* ``prefix``: the same for a batch whose requests share a long prefix, which is read once for all of them.

``requests`` requests take part in a step.  The longest has ``context`` tokens when the step is done, ``tokens`` of them new;
``spread`` says how the others lie below that: all alike ("even") or over the logarithm ("log").  ``block`` is the number of
tokens in a block of the cache.  ``layout`` names the order of a cache in memory: "head" [blocks, heads, block, ...] or "token"
[blocks, block, heads, ...]; ``fused`` says that q, k and v are columns of one product's output.
"""
import math

import torch

own = False

FLOPS = 4 * 128 * 32 * 8192 * 8193 // 2     # the largest listed attention; drawn ones stay within these figures
ROWS = 2 * 16 * 32768 * 8 * 128             # values of the longest contexts, keys and values together
SCORES = 32 * 8192 * 8192                   # scores that the plain form holds at once
NEW = 2 * 8192 * 8 * 128                    # values that a step stores

EXPONENTS = {"float16": (-23, 13), "bfloat16": (-125, 125)}
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _case(name, op, **more):
    case = {"name": name, "op": op, "dtype": "float16", "heads": 32, "kv_heads": 8, "dim": 128, "block": 16, "requests": 1,
            "context": 1, "tokens": 1, "spread": "even", "window": 0, "sinks": 0, "prefix": 0, "layout": "head",
            "fused": False}
    case.update(more)
    return case


def listed():
    return [
        # keys and values of a decoding step of a batch, and of a long prompt out of a fused q/k/v product
        _case("store-decode-64", "store", requests=64, context=1024, spread="log"),
        _case("store-prompt-8192", "store", dtype="bfloat16", context=8192, tokens=8192, fused=True),
        # a short conversation and a long document on their way to another process, or to attention of one's own; narrow odd heads
        _case("read-333-dim80", "read", context=333, dim=80, block=24),
        _case("read-32768", "read", dtype="bfloat16", context=32768, block=64),
        # decoding: one short conversation, where latency counts; a batch of long ones under a window with sinks, whose
        # blocks behind the window were given back; a batch of long documents, the call that is bound by memory
        _case("decode-1x512", "attend", context=512),
        _case("decode-64-window4096", "attend", dtype="bfloat16", requests=64, context=32768, spread="log", window=4096, sinks=4, block=64),
        _case("decode-16x32768", "attend", requests=16, context=32768, block=64),
        # drafts of five tokens a request, heads in sevens
        _case("drafts-24x5-dim64", "attend", heads=14, kv_heads=2, dim=64, requests=24, context=6001, tokens=5, spread="log"),
        # prompts: a long one; pieces of prompts of ragged lengths behind contexts that are in the cache, narrow heads in sevens,
        # blocks that are no power of two
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
    op = rng.choice(("store", "store", "read", "attend", "attend", "attend", "attend", "attend", "prefix", "prefix"))
    kv_heads = rng.choice((1, 2, 4, 8, 8, 8, 16, 32))
    group = rng.choice([g for g in (1, 1, 4, 4, 5, 7, 8, 16) if g * kv_heads <= 64])
    c = {"op": op, "dtype": rng.choice(("float16", "float16", "bfloat16")), "heads": group * kv_heads, "kv_heads": kv_heads,
         "dim": rng.choice((64, 128, 128, 128, 80, 96, 256, 72)), "block": rng.choice((16, 16, 32, 64, 128, 24, 7)),
         "requests": 1 if op == "read" else _log(rng, 1, 256), "context": _log(rng, 16, 32768), "tokens": 1,
         "spread": rng.choice(("even", "log", "log")), "window": 0, "sinks": 0, "prefix": 0,
         "layout": rng.choice(("head", "head", "token")), "fused": rng.random() < 0.3}
    if op == "store" and rng.random() < 0.6 or op == "attend" and rng.random() < 0.5:
        c["tokens"] = _log(rng, 1, min(c["context"], 8192))     # prompts, or pieces of them
    if op == "attend" and rng.random() < 0.5:
        c["window"], c["sinks"] = _log(rng, 64, 8192), rng.choice((0, 1, 4, 33))
    if op == "prefix":
        c["prefix"], c["context"] = _log(rng, 128, 32768), _log(rng, 1, 4096)
        if rng.random() < 0.3:
            c["tokens"] = _log(rng, 1, min(c["context"], 16))

    def fits():
        b, values = c["requests"], 2 * c["kv_heads"] * c["dim"]
        seen = _width(c) + c["prefix"]
        held = sum(-(-x // c["block"]) * c["block"] for x, _ in _lengths(c))
        if op in ("store", "read"):
            return sum(n for _, n in _lengths(c)) * values <= NEW and held * values <= ROWS
        return work(c)["flops"] <= FLOPS and b * seen * values <= ROWS and b * c["heads"] * c["tokens"] * seen <= SCORES
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


def _row_bytes(case):
    """(codes, scales) of a head's row."""
    groups = -(-case["dim"] // 32)
    return 16 * groups, 2 if groups <= 2 else 4 if groups <= 4 else 8


def work(case):
    lengths = _lengths(case)
    T = sum(n for _, n in lengths)
    D, hq, hk = case["dim"], case["heads"], case["kv_heads"]
    row = D / 2 + D / 32                     # what the format takes for a head's values of a token
    if case["op"] == "store":                # values in, rows and what they stand for out
        return {"bytes": int(2 * T * hk * (2 * D + row + 2 * D)) + 4 * T, "flops": 0}
    if case["op"] == "read":
        return {"bytes": int(2 * case["context"] * hk * (row + 2 * D)) + 4 * case["context"], "flops": 0}
    rows = sum(s + c - lo for c, n in lengths for s, lo in [_seen(case, c, n)]) + case["prefix"]
    pairs = sum(_pairs(case, c, n) for c, n in lengths) + T * case["prefix"]
    return {"bytes": int(2 * rows * hk * row) + 2 * 2 * T * hq * D + 4 * (rows // case["block"] + 2 * len(lengths)),
            "flops": 4 * pairs * hq * D}


# ------------------------------------------------------------------ the format, in elementary operations
def _encode(x, dtype):
    """Rows [..., dim] as (codes, scales): bytes [..., 16 groups] and [..., groups]."""
    D = x.shape[-1]
    x = torch.nn.functional.pad(x.float(), (0, -D % 32)).unflatten(-1, (-1, 32))
    size = x.abs()
    most = size.amax(-1, keepdim=True)
    fine = torch.isfinite(size).all(-1, keepdim=True)
    most = torch.where(fine, most, 1.0)
    # exponent bits; a mantissa of 1.75 or more carries into them
    e = (((most.view(torch.int32) + 0x200000) >> 23) - 129).clamp(*EXPONENTS[str(dtype).split(".")[1]])
    m = size * ((127 - e) << 23).view(torch.float32)
    code = ((m > 0.25).to(torch.uint8) + (m >= 0.75) + (m > 1.25) + (m >= 1.75) + (m > 2.5) + (m >= 3.5) + (m > 5.0))
    code = torch.where(fine, code | ((x < 0).to(torch.uint8) << 3), 0).flatten(-2)
    return code[..., ::2] | (code[..., 1::2] << 4), torch.where(fine, e + 127, 255).to(torch.uint8).flatten(-2)


def _decode(codes, scales, dim):
    """The values of rows of bytes, in 32 bits."""
    table = torch.tensor(VALUES + tuple(-v for v in VALUES), device=codes.device)
    scales = scales[..., :codes.shape[-1] // 16].int()
    power = torch.where(scales == 255, float("nan"), (scales << 23).view(torch.float32))
    values = torch.stack((table[(codes & 15).int()], table[(codes >> 4).int()]), -1).flatten(-2)
    return (values.unflatten(-1, (-1, 32)) * power[..., None]).flatten(-2)[..., :dim]


# ------------------------------------------------------------------ inputs
def _empty_cache(case, blocks):
    """Codes and scales of keys and of values; unwritten slots hold whatever was there."""
    b, h = case["block"], case["kv_heads"]
    made = []
    for n, bits in zip(_row_bytes(case), (0x7A, 255)):
        shape = (2, blocks, b, h, n) if case["layout"] == "token" else (2, blocks, h, b, n)
        both = torch.full(shape, bits, dtype=torch.uint8, device="cuda")
        made.append(both if case["layout"] == "token" else both.transpose(2, 3))
    return made[0][0], made[0][1], made[1][0], made[1][1]


def _filled_cache(case, blocks, dtype, gen):
    """Keys with a few channels of larger size, as rotated keys have them, and values."""
    kc, vc, ks, vs = _empty_cache(case, blocks)
    D, groups = case["dim"], _row_bytes(case)[0] // 16
    step = max(1, 2 ** 25 // (case["block"] * case["kv_heads"] * D))
    for b0 in range(0, blocks, step):
        n = min(step, blocks - b0)
        for codes, scales, keys in ((kc, ks, True), (vc, vs, False)):
            x = torch.randn((n, case["block"], case["kv_heads"], D), device="cuda", generator=gen, dtype=dtype)
            if keys:
                x[..., ::29] *= 3
            c, s = _encode(x, dtype)
            codes[b0:b0 + n], scales[b0:b0 + n, ..., :groups] = c, s
    return kc, vc, ks, vs


def _new(case, T, dtype, gen):
    """q, k and v of a step's tokens."""
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if case["fused"]:
        qkv = torch.randn((T, (hq + 2 * hk) * d), device="cuda", generator=gen, dtype=dtype)
        q, k, v = (x.view(T, -1, d) for x in qkv.split((hq * d, hk * d, hk * d), dim=1))
    else:
        q, k, v = (torch.randn((T, h, d), device="cuda", generator=gen, dtype=dtype) for h in (hq, hk, hk))
    k[..., ::29] *= 3
    return q, k, v


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, blk = getattr(torch, case["dtype"]), case["block"]
    lengths = _lengths(case)
    T = sum(n for _, n in lengths)
    most = max(c for c, _ in lengths)
    wide = -(-most // blk) + 3                                   # the tables have room for what comes
    state = {"case": case, "dtype": dtype, "T": T, "most": most, "seen": _width(case), "tokens": max(n for _, n in lengths)}
    if case["op"] in ("store", "read"):
        blocks = sum(-(-c // blk) for c, _ in lengths) + 3
        order = torch.randperm(blocks, device="cuda", generator=gen)
        slots, at = [], 0
        for c, n in lengths:
            p = torch.arange(c - n if case["op"] == "store" else 0, c, device="cuda")
            slots.append(order[at + p // blk] * blk + p % blk)
            at += -(-c // blk)
        state["slots"] = torch.cat(slots).to(torch.int32)
        if case["op"] == "store":
            _, state["k"], state["v"] = _new(case, T, dtype, gen)
            state["cache"] = _empty_cache(case, blocks)
        else:
            state["cache"] = _filled_cache(case, blocks, dtype, gen)
        return state
    # blocks that no new token sees, behind a window, were given back: the tables hold -1 there
    kept = [[j for j in range(-(-c // blk)) if j * blk < s or (j + 1) * blk > lo] for c, n in lengths for s, lo in [_seen(case, c, n)]]
    shared = -(-case["prefix"] // blk)
    blocks = sum(map(len, kept)) + shared + 3
    order = torch.randperm(blocks, device="cuda", generator=gen).to(torch.int32)
    cache = _filled_cache(case, blocks, dtype, gen)
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
            for scales in cache[2:]:
                scales[block, used:] = 255
    starts = [0]
    for _, n in lengths:
        starts.append(starts[-1] + n)
    q, _, _ = _new(case, T, dtype, gen)
    state.update(q=q.mul_(2), cache=cache, tables=tables, starts=_ints(starts), contexts=_ints([c for c, _ in lengths]),
                 shared=order[:shared].clone())
    return state


# ------------------------------------------------------------------ the framework's calls
def _own(state):
    from autogptq.tvm_amd import attention

    c, s = state["case"], state
    k_codes, v_codes, k_scales, v_scales = s["cache"]
    k_cache, v_cache = attention.Mxfp4(k_codes, k_scales), attention.Mxfp4(v_codes, v_scales)
    if c["op"] == "store":
        attention.cache_write(s["k"], s["v"], k_cache, v_cache, s["slots"])
    if c["op"] in ("store", "read"):
        return attention.cache_read(k_cache, v_cache, s["slots"], c["dim"], s["dtype"])
    if c["op"] == "attend":
        return attention.paged_attention(s["q"], k_cache, v_cache, s["tables"], s["starts"], s["contexts"],
                                         max_context=s["most"], window=c["window"], sinks=c["sinks"])
    return attention.shared_prefix_attention(s["q"], k_cache, v_cache, s["shared"], c["prefix"], s["tables"],
                                             s["starts"], s["contexts"], max_context=s["most"])


# ------------------------------------------------------------------ the plain forms
def _plain_store(s):
    blk, groups = s["case"]["block"], _row_bytes(s["case"])[0] // 16
    block, at = s["slots"] // blk, s["slots"] % blk
    for x, codes, scales in zip((s["k"], s["v"]), s["cache"][:2], s["cache"][2:]):
        codes[block, at], scales[..., :groups][block, at] = _encode(x, s["dtype"])


def _plain_read(s):
    blk, D = s["case"]["block"], s["case"]["dim"]
    block, at = s["slots"] // blk, s["slots"] % blk
    return [_decode(codes[block, at], scales[block, at], D).to(s["dtype"]) for codes, scales in zip(s["cache"][:2], s["cache"][2:])]


def _owner(starts, T):
    return torch.searchsorted(starts[1:].contiguous(), torch.arange(T, dtype=torch.int32, device=starts.device), right=True)


def _rows(s, which, tables, at, there):
    """The rows of the keys (0) or values (1) at the positions `at` of every request, [requests, heads, positions, dim] in 32
    bits; zeros where there is none."""
    codes, scales, blk = s["cache"][which], s["cache"][2 + which], s["case"]["block"]
    block = torch.where(there, torch.gather(tables, 1, torch.where(there, at // blk, 0).long()), 0)
    slot = torch.where(there, at % blk, 0)
    rows = _decode(codes[block, slot], scales[block, slot], s["case"]["dim"])
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
    keys, values = (_rows(s, n, s["tables"], at, there) for n in (0, 1))
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
        keys0, values0 = (_rows(s, n, s["shared"][None], j, all_there)[0] for n in (0, 1))
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
    if op == "store":
        _plain_store(state)
    return _plain_read(state) if op in ("store", "read") else _plain_attend(state)


# ------------------------------------------------------------------ the definition, in 64 bits
def _stored(x, dtype):
    """What rows stand for once they are in the cache."""
    D = x.shape[-1]
    low, high = EXPONENTS[str(dtype).split(".")[1]]
    x = torch.nn.functional.pad(x.double(), (0, -D % 32)).unflatten(-1, (-1, 32))
    part, power = torch.frexp(x.abs().amax(-1, keepdim=True))        # part in [1/2, 1)
    power = torch.ldexp(torch.ones_like(part), (power - 3 + (part >= 0.875)).clamp(low, high))
    at = x.abs() / power
    best, off = torch.zeros_like(at), torch.full_like(at, math.inf)
    for code in (0, 2, 4, 6, 1, 3, 5, 7):                            # (the even ones first: they keep their ties)
        d = (at - VALUES[code]).abs()
        best, off = torch.where(d < off, VALUES[code], best), torch.minimum(d, off)
    return (best * power * torch.sign(x)).flatten(-2)[..., :D]


def _meant(codes, scales, dim):
    """The values of rows of a cache."""
    values = torch.tensor(VALUES, dtype=torch.float64, device=codes.device)
    out = torch.empty((*codes.shape[:-1], 2 * codes.shape[-1]), dtype=torch.float64, device=codes.device)
    for half, code in ((0, codes % 16), (1, codes // 16)):
        out[..., half::2] = values[(code % 8).long()] * (1.0 - 2.0 * (code // 8).double())
    group = torch.arange(out.shape[-1], device=codes.device) // 32
    power = torch.exp2(scales.double() - 127.0)
    return (out * torch.where(scales == 255, math.nan, power)[..., group])[..., :dim]


def exact(case, seed):
    s, blk, lengths, D = prepare(case, seed), case["block"], _lengths(case), case["dim"]
    if case["op"] == "store":
        return [_stored(s[n], s["dtype"]) for n in ("k", "v")]
    rows = lambda which, block, at: _meant(s["cache"][which][block, at], s["cache"][2 + which][block, at], D)
    if case["op"] == "read":
        slots = s["slots"].long()
        return [rows(which, slots // blk, slots % blk) for which in (0, 1)]
    T, hq, _ = s["q"].shape
    hk, w = case["kv_heads"], case["window"]
    out = torch.zeros((T, hq, D), dtype=torch.float64, device="cuda")
    j = torch.arange(case["prefix"], device="cuda")
    prefix = s["shared"].long()[j // blk]
    k0, v0 = (rows(which, prefix, j % blk) for which in (0, 1))
    begin = 0
    for b, (c, n) in enumerate(lengths):
        seen_first, lo = _seen(case, c, n)
        at = torch.cat([torch.arange(seen_first, device="cuda"), torch.arange(lo, c, device="cuda")])
        block = s["tables"][b].long()[at // blk]
        k = torch.cat([k0, rows(0, block, at % blk)])
        v = torch.cat([v0, rows(1, block, at % blk)])
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
