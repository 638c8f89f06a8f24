"""A paged key/value cache for the decoders whose linear layers this package holds, and the attention that reads it.

The reference leaves attention to the model (auto_gptq/modeling/_base.py:478-569 loads a ``transformers`` model whose linear
layers are replaced); here a serving step finds what stands between q/k/v and o as operators of their own:

* ``cache_tables``             block tables, slot maps, query offsets and positions of a step, from the requests' lengths
* ``cache_write``              the step's keys and values into their slots
* ``paged_attention``          causal attention over the requests' blocks: prompts, pieces of prompts and single tokens, mixed
                               as they come, with or without a sliding window and first tokens that stay visible (sinks)
* ``shared_prefix_attention``  the same for requests behind one long prefix, which is read once for all of them

All run on the current stream of the tensors' device, have no backward, and exist as ``torch.ops.gptq_hip.*`` too.  They can be
captured by ``torch.cuda.graph``: a capture gets a workspace of its own from the graph's memory, whatever runs before or after it
(the graph clears its counters, one small launch a replay); what the kernels need loaded, a call on any stream before it loads.  Caches are float16 or bfloat16
[blocks, block_size, kv_heads, dim] in any order of memory whose last dimension is contiguous; dim is a multiple of 8 up to 256.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import ops


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


def cache_write(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor) -> None:
    """``k`` and ``v`` [tokens, kv_heads, dim] (columns of a fused product as they are) into ``slots`` of the cache; tokens
    with slot -1 are skipped."""
    _call("cache_write", k, v, k_cache, v_cache, slots)


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, tables: torch.Tensor, starts: torch.Tensor,
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
    return _call("paged_attention", q, k_cache, v_cache, tables, starts, contexts, max_context, window, sinks, _scale(scale))


def shared_prefix_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, prefix_blocks: torch.Tensor,
                            prefix_length: int, tables: torch.Tensor, starts: torch.Tensor, contexts: torch.Tensor, *,
                            max_context: int = 0, scale: Optional[float] = None) -> torch.Tensor:
    """``paged_attention`` where every request stands behind the same ``prefix_length`` tokens, whose blocks are
    ``prefix_blocks``: all tokens see all of them, and they are read once for the batch.  ``tables``, ``contexts`` and
    ``max_context`` count a request's own tokens only."""
    return _call("shared_prefix_attention", q, k_cache, v_cache, prefix_blocks, prefix_length, tables, starts, contexts,
                 max_context, _scale(scale))


def _scale(scale: Optional[float]) -> float:
    if scale is None:
        return 0.0      # (the operators' word for 1 / sqrt(dim))
    if not scale > 0:
        raise ValueError(f"scale must be positive, got {scale}")
    return scale


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


__all__ = ["CacheTables", "cache_tables", "cache_write", "paged_attention", "shared_prefix_attention"]
