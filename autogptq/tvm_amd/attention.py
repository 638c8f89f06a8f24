"""A paged key/value cache for the decoders whose linear layers this package holds, and the attention that reads it.

The reference leaves attention to the model (auto_gptq/modeling/_base.py:478-569 loads a ``transformers`` model whose linear
layers are replaced); here a serving step finds what stands between q/k/v and o as operators of their own:

* ``cache_tables``             block tables, slot maps, query offsets and positions of a step, from the requests' lengths
* ``cache_write``              the step's keys and values into their slots
* ``cache_read``               the rows of slots back
* ``paged_attention``          causal attention over the requests' blocks: prompts, pieces of prompts and single tokens, mixed
                               as they come, with or without a sliding window and first tokens that stay visible (sinks)
* ``shared_prefix_attention``  the same for requests behind one long prefix, which is read once for all of them

All run on the current stream of the tensors' device, have no backward, and exist as ``torch.ops.gptq_hip.*`` too.  They can be
captured by ``torch.cuda.graph``: a capture gets a workspace of its own from the graph's memory, whatever runs before or after it
(the graph clears its counters, one small launch a replay); what the kernels need loaded, a call on any stream before it loads.  Caches are float16 or bfloat16
[blocks, block_size, kv_heads, dim] in any order of memory whose last dimension is contiguous; dim is a multiple of 8 up to 256.

A cache may also be held in MXFP4, 4.25 bits a value where dim is 64, 128 or 256: pass an ``Mxfp4`` (see there, and ``mxfp4_cache``) wherever a cache is asked for; the
write quantises, the attention reads the codes.  The operators of these are ``torch.ops.gptq_hip.<name>_mx``, with codes and scales as
two arguments each.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple, Union

import torch

from . import ops


class Mxfp4(NamedTuple):
    """Keys or values of a cache in MXFP4, the microscaling format with 4-bit floats.  A head's ``dim`` values of a token, padded to
    a multiple of 32, are groups of 32 codes and a power of two 2^e each; a code is a sign and one of 0, 1/2, 1, 3/2, 2, 3, 4, 6.
    A write takes the e that puts a group's largest magnitude into [3.5, 7) 2^e and the nearest codes, ties to the even one (a group of
    float16 values has e within -23 .. 13, of bfloat16 -125 .. 125: what it stands for is a value of the type, and what lies beyond 6 2^e
    becomes that).  A group with an infinity or a NaN stands for NaN.  A cache is read in the type it was written in."""

    codes: torch.Tensor       # uint8 [blocks, block_size, kv_heads, 16 ceil(dim / 32)]: value 2 j in the low half of byte j
    scales: torch.Tensor      # uint8 [blocks, block_size, kv_heads, 2 (dim up to 64), 4 (up to 128) or 8]: e + 127; 255: NaN


Cache = Union[torch.Tensor, Mxfp4]


def mxfp4_cache(blocks: int, block_size: int, kv_heads: int, dim: int, device="cuda:0") -> Tuple[Mxfp4, Mxfp4]:
    """Keys and values of a cache in MXFP4, unwritten.  (A block's rows of a head lie together: whole lines for the kernels that read one
    head.)"""
    if dim < 8 or dim % 8 or dim > 256:
        raise ValueError(f"dim must be a multiple of 8 up to 256, got {dim}")
    codes, scales = (torch.empty((2, blocks, kv_heads, block_size, n), dtype=torch.uint8, device=device).transpose(2, 3)
                     for n in (-(-dim // 32) * 16, 2 if dim <= 64 else 4 if dim <= 128 else 8))
    return Mxfp4(codes[0], scales[0]), Mxfp4(codes[1], scales[1])


class CacheTables(NamedTuple):
    """What ``cache_tables`` returns, int32 on the GPU."""

    starts: torch.Tensor      # [requests + 1]  new tokens before each request, and all of them
    contexts: torch.Tensor    # [requests]      tokens in the cache when the step's are written
    slots: torch.Tensor       # [tokens]        slot of every new token, -1 where there is none
    positions: torch.Tensor   # [tokens]        its position in its request
    taken: torch.Tensor       # [1]             blocks needed from the free list


def cache_tables(lengths: torch.Tensor, counts: torch.Tensor, tables: torch.Tensor, free_blocks: torch.Tensor, tokens: int,
                 block_size: int) -> CacheTables:
    """The bookkeeping of a step in one launch: request b has ``lengths[b]`` tokens in the cache and gets ``counts[b]`` more
    (int32, on the GPU).  The blocks these need come from the front of ``free_blocks``, requests in order, and are entered
    into ``tables`` [requests, width] in place.  ``tokens`` is the sum of the counts, which the caller knows without asking
    the GPU.  If ``taken`` exceeds ``free_blocks``, or a table its width, the tokens that found no place have slot -1."""
    return CacheTables(*_call("cache_tables", lengths, counts, tables, free_blocks, tokens, block_size))


def cache_write(k: torch.Tensor, v: torch.Tensor, k_cache: Cache, v_cache: Cache, slots: torch.Tensor) -> None:
    """``k`` and ``v`` [tokens, kv_heads, dim] (columns of a fused product as they are) into ``slots`` of the cache; tokens
    with slot -1 are skipped.  Slots are distinct (one that is named twice is left with parts of both tokens)."""
    if _packed(k_cache, v_cache):
        _call("cache_write_mx", k, v, *k_cache, *v_cache, slots)
    else:
        _call("cache_write", k, v, k_cache, v_cache, slots)


def cache_read(k_cache: Cache, v_cache: Cache, slots: torch.Tensor, dim: Optional[int] = None,
               dtype: Optional[torch.dtype] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(k, v) [tokens, kv_heads, dim]: the rows of ``slots`` (int32), zeros for slots that the cache does not have (-1).  ``dim`` and
    ``dtype`` say what an ``Mxfp4`` cache was written with (default: all of its groups, float16); other caches know both."""
    if _packed(k_cache, v_cache):
        dim = 2 * k_cache.codes.shape[-1] if dim is None else dim
        return _call("cache_read_mx", *k_cache, *v_cache, slots, dim, dtype or torch.float16)
    if dim not in (None, k_cache.shape[-1]) or dtype not in (None, k_cache.dtype):
        raise ValueError(f"the cache holds rows of {k_cache.shape[-1]} in {k_cache.dtype}, not of {dim} in {dtype}")
    return _call("cache_read", k_cache, v_cache, slots)


def paged_attention(q: torch.Tensor, k_cache: Cache, v_cache: Cache, tables: torch.Tensor, starts: torch.Tensor,
                    contexts: torch.Tensor, *, max_context: int = 0, window: int = 0, sinks: int = 0,
                    scale: Optional[float] = None) -> torch.Tensor:
    """[tokens, heads, dim]: the attention of the step's tokens.  Request b has the tokens ``starts[b] .. starts[b + 1]``, the
    last of them at position ``contexts[b] - 1`` (their keys are in the cache already); a token at position i sees the
    positions j <= i, under a ``window`` only j > i - window and the first ``sinks``.  Blocks that no token of a request
    sees may be given back: their table entries are not read, nor are slots past a context.  Values are finite up to a request's
    last token (one that a token does not see may still count for it, with the share 0).  A token that sees nothing gets zeros, and so do
    tokens of no request (those from ``starts[-1]`` on: a step may be padded to a fixed size).  Query head n reads
    key/value head n // (heads / kv_heads).  ``max_context``: the longest context as the host knows it, by which the work is
    divided (0: the tables' width); results do not depend on it beyond the order of sums.  ``scale``: 1 / sqrt(dim) if None."""
    if _packed(k_cache, v_cache):
        return _call("paged_attention_mx", q, *k_cache, *v_cache, tables, starts, contexts, max_context, window, sinks, _scale(scale))
    return _call("paged_attention", q, k_cache, v_cache, tables, starts, contexts, max_context, window, sinks, _scale(scale))


def shared_prefix_attention(q: torch.Tensor, k_cache: Cache, v_cache: Cache, prefix_blocks: torch.Tensor,
                            prefix_length: int, tables: torch.Tensor, starts: torch.Tensor, contexts: torch.Tensor, *,
                            max_context: int = 0, scale: Optional[float] = None) -> torch.Tensor:
    """``paged_attention`` where every request stands behind the same ``prefix_length`` tokens, whose blocks are
    ``prefix_blocks``: all tokens see all of them, and they are read once for the batch.  ``tables``, ``contexts`` and
    ``max_context`` count a request's own tokens only."""
    if _packed(k_cache, v_cache):
        return _call("shared_prefix_attention_mx", q, *k_cache, *v_cache, prefix_blocks, prefix_length, tables, starts, contexts,
                     max_context, _scale(scale))
    return _call("shared_prefix_attention", q, k_cache, v_cache, prefix_blocks, prefix_length, tables, starts, contexts,
                 max_context, _scale(scale))


def _scale(scale: Optional[float]) -> float:
    if scale is None:
        return 0.0      # (the operators' word for 1 / sqrt(dim))
    if not scale > 0:
        raise ValueError(f"scale must be positive, got {scale}")
    return scale


def _packed(k_cache: Cache, v_cache: Cache) -> bool:
    packed = isinstance(k_cache, Mxfp4)
    if packed != isinstance(v_cache, Mxfp4):
        raise TypeError("k_cache and v_cache must both be tensors or both be Mxfp4")
    return packed


def _call(name: str, *args):
    """The operator by its C function (csrc/python_call.cpp), or by torch.ops where that leaves it to the dispatcher."""
    if not ops.NATIVE_OPS:
        raise RuntimeError("the operator library is missing or stale: build it with `python -m autogptq.tvm_amd.build` "
                           "(there is no fallback path)")
    if not torch.compiler.is_compiling():
        result = getattr(ops.CALL, name)(*args)
        if result is not NotImplemented:
            return result
    return getattr(torch.ops.gptq_hip, name)(*args)


__all__ = ["CacheTables", "Mxfp4", "cache_read", "cache_tables", "cache_write", "mxfp4_cache", "paged_attention", "shared_prefix_attention"]
