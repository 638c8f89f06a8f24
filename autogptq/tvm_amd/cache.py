"""``PagedCache``: the blocks of a paged key/value cache, whose they are, and the operators of ``attention.py`` on them.

The host keeps the requests' lengths (a serving program knows how many tokens it hands in), so nothing here waits for the
GPU: whether the blocks suffice is known before a launch, and block tables, slot maps and the list of free blocks stay on
the GPU."""
from __future__ import annotations

from typing import List, NamedTuple, Optional, Sequence, Tuple

import torch

from . import attention


class Step(NamedTuple):
    """One step of some requests: what ``PagedCache.step`` returns and ``write`` and ``attend`` take, for every layer.  It stays as it is
    whatever is trimmed or freed between two layers; blocks that were given back hold what they held until a later step's ``write``."""

    tables: torch.Tensor      # [requests, width]
    starts: torch.Tensor      # [requests + 1]
    contexts: torch.Tensor    # [requests]
    slots: torch.Tensor       # [tokens]
    positions: torch.Tensor   # [tokens], for rotary embeddings and the like
    max_context: int
    prefix: Optional[Tuple[torch.Tensor, int]]     # blocks and length of a prefix that all of them share
    window: int = 0           # the widest window, and the most sinks, under which the blocks that trim() has given back are not
    sinks: int = 0            # seen (window 0: none are missing)


class PagedCache:
    """``blocks`` blocks of ``block_size`` tokens in ``layers`` layers, for up to ``max_requests`` requests at a time, each of up to
    ``max_context`` tokens.  A request is a number below ``max_requests``; it exists from its first ``step`` to ``free``."""

    def __init__(self, layers: int, blocks: int, block_size: int, kv_heads: int, dim: int, max_requests: int, max_context: int,
                 dtype=torch.float16, device="cuda:0"):
        self.block_size = block_size
        # a block's keys (or values) of a head lie together: whole kilobytes for the kernels that read one head
        both = torch.empty((layers, 2, blocks, kv_heads, block_size, dim), dtype=dtype, device=device).transpose(3, 4)
        self.k, self.v = both[:, 0], both[:, 1]
        width = -(-max_context // block_size)
        self.tables = torch.full((max_requests, width), -1, dtype=torch.int32, device=device)
        self._free = torch.arange(blocks, dtype=torch.int32, device=device)
        self._lengths = [0] * max_requests                  # the host's, and the same on the GPU
        self._on_gpu = torch.zeros(max_requests, dtype=torch.int32, device=device)
        self._prefixes: List[Optional[Tuple[torch.Tensor, int]]] = [None] * max_requests
        self._source: List[Optional[int]] = [None] * max_requests       # whose prefix that is
        self._kept = [(0, 0)] * max_requests                # blocks [a, b) of a request that trim() has given back
        self._rows = ((), None)                             # the requests of the last step, as a tensor
        self._handed_out = False                            # whether a Step holds self.tables itself, or a row as its prefix

    @property
    def free_blocks(self) -> int:
        return self._free.numel()

    def length(self, request: int) -> int:
        """Tokens of a request in the cache (its own: without those of a shared prefix)."""
        self._known(request)
        return self._lengths[request]

    def _known(self, *requests: int) -> None:
        for r in requests:
            if not 0 <= r < len(self._lengths):
                raise IndexError(f"request {r} is not a number from 0 to {len(self._lengths) - 1}")

    def _blocks(self, tokens: int) -> int:
        return -(-tokens // self.block_size)

    def share(self, source: int, request: int) -> None:
        """``request`` (without tokens so far) stands behind the tokens that ``source`` has now, whose blocks it reads and does
        not own: ``source`` is neither trimmed nor freed while others stand behind it.  (What it gets later they do not see.)"""
        self._known(source, request)
        if self._lengths[request] or self._prefixes[request] is not None:
            raise ValueError(f"request {request} has tokens already")
        if self._prefixes[source] is not None or self._kept[source] != (0, 0):
            raise ValueError(f"request {source} stands behind a prefix itself, or was trimmed")
        n = self._lengths[source]
        if n:
            self._prefixes[request], self._source[request] = (self.tables[source, :self._blocks(n)], n), source
            self._handed_out = True

    def _alone(self, request: int) -> None:
        behind = [r for r, s in enumerate(self._source) if s == request]
        if behind:
            raise ValueError(f"requests {behind} stand behind the tokens of request {request}")

    def step(self, requests: Sequence[int], counts: Sequence[int]) -> Step:
        """Makes room for ``counts[i]`` more tokens of ``requests[i]``.  Raises before anything is launched if there is none."""
        requests = tuple(requests)
        self._known(*requests)
        if len(set(requests)) != len(requests) or len(requests) != len(counts) or min(counts, default=0) < 0:
            raise ValueError("requests must be distinct, with a count of at least 0 each")
        prefixes = [self._prefixes[r] for r in requests]
        if len({(self._source[r], p[1]) if p else None for r, p in zip(requests, prefixes)}) > 1:
            raise ValueError("the requests of a step must stand behind one prefix, or all behind none")
        after = [self._lengths[r] + n for r, n in zip(requests, counts)]
        gaps = [(self._lengths[r] + 1 - self._kept[r][1] * self.block_size, self._kept[r][0] * self.block_size)
                for r, n in zip(requests, counts) if n and self._kept[r][1]]
        if max(after, default=0) > self.tables.shape[1] * self.block_size:
            raise RuntimeError(f"a request of {max(after)} tokens does not fit the tables")
        need = sum(self._blocks(a) - self._blocks(self._lengths[r]) for r, a in zip(requests, after))
        if need > self.free_blocks:
            raise RuntimeError(f"{need} blocks are needed and {self.free_blocks} are free")
        device = self.tables.device
        if self._rows[0] != requests:
            self._rows = (requests, torch.tensor(requests, dtype=torch.int64, device=device))
        rows = self._rows[1]
        every = requests == tuple(range(self.tables.shape[0]))
        tables = self.tables if every else self.tables[rows]
        self._handed_out |= every
        made = attention.cache_tables(self._on_gpu[rows], torch.tensor(counts, dtype=torch.int32).to(device, non_blocking=True), tables,
                                      self._free, sum(counts), self.block_size)
        if not every:
            self.tables[rows] = tables
        self._on_gpu[rows] = made.contexts
        self._free = self._free[need:]
        for r, a in zip(requests, after):
            self._lengths[r] = a
        prefix = prefixes[0] if prefixes else None
        return Step(tables, made.starts, made.contexts, made.slots, made.positions + prefix[1] if prefix else made.positions,
                    max(after, default=0), prefix, min((w for w, _ in gaps), default=0), min((k for _, k in gaps), default=0))

    def write(self, layer: int, k: torch.Tensor, v: torch.Tensor, step: Step) -> None:
        """The step's keys and values [tokens, kv_heads, dim] of a layer."""
        attention.cache_write(k, v, self.k[layer], self.v[layer], step.slots)

    def attend(self, layer: int, q: torch.Tensor, step: Step, window: int = 0, sinks: int = 0,
               scale: Optional[float] = None) -> torch.Tensor:
        """The attention of the step's queries [tokens, heads, dim] in a layer, after ``write``."""
        k, v = self.k[layer], self.v[layer]
        if step.window and not (0 < window <= step.window and sinks <= step.sinks):
            raise ValueError(f"what trim has left of these requests suffices for windows of at most {step.window} tokens and {step.sinks} "
                             f"sinks, not for window={window}, sinks={sinks}")
        if step.prefix is None:
            return attention.paged_attention(q, k, v, step.tables, step.starts, step.contexts, max_context=step.max_context,
                                             window=window, sinks=sinks, scale=scale)
        if window:
            raise NotImplementedError("a sliding window behind a shared prefix")
        return attention.shared_prefix_attention(q, k, v, step.prefix[0], step.prefix[1], step.tables, step.starts, step.contexts,
                                                 max_context=step.max_context, scale=scale)

    def _forget(self, request: int, first: int, last: Optional[int] = None) -> None:
        """Takes entries out of a request's table.  (Steps keep theirs; the entries that later steps add lie past their contexts.)"""
        if self._handed_out:
            self.tables, self._handed_out = self.tables.clone(), False
        self.tables[request, first:last] = -1

    def trim(self, request: int, window: int, sinks: int = 0) -> int:
        """Gives back the blocks that no later token of a request sees under a window (of at least 1) with sinks; returns how
        many.  From then on the request is attended to with this window and these sinks, or narrower ones (what sees blocks that are
        gone is refused)."""
        self._known(request)
        if window < 1:
            raise ValueError("trim needs a window")
        if self._prefixes[request] is not None:
            raise NotImplementedError("a sliding window behind a shared prefix")
        self._alone(request)
        first, last = self._blocks(sinks), max(0, self._lengths[request] + 1 - window) // self.block_size
        start, gone = self._kept[request]
        if gone > 0 and first > start:
            raise ValueError(f"request {request} has kept its first {start * self.block_size} tokens only: {sinks} sinks are too many")
        first = max(first, gone)
        if last <= first:
            return 0
        self._free = torch.cat([self._free, self.tables[request, first:last]])
        self._forget(request, first, last)
        self._kept[request] = (start if gone > 0 else first, last)
        return last - first

    def free(self, request: int) -> None:
        """Ends a request: its blocks are free again."""
        self._known(request)
        self._alone(request)
        a, b = self._kept[request]
        n = self._blocks(self._lengths[request])
        self._free = torch.cat([self._free, self.tables[request, :a], self.tables[request, b:n]])
        self._forget(request, 0)
        self._on_gpu[request] = 0
        self._lengths[request], self._kept[request] = 0, (0, 0)
        self._prefixes[request] = self._source[request] = None


__all__ = ["PagedCache", "Step"]
