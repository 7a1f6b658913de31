"""A paged key / value cache: one pool of pages for all layers, sequences as lists of pages.

``PagedCache`` keeps the books on the host (which page belongs to whom, how often it is shared) and
touches the device only where pages are copied: a fork shares its pages and copies the last one,
if it is partly filled, when one of the two first writes to it; ``compact`` moves pages down.
``step`` turns "these sequences get so many new tokens" into the index tensors that
``rope_append`` and ``paged_attention`` take.
"""
from __future__ import annotations

import heapq
from dataclasses import dataclass
from typing import Dict, List, Optional, Sequence, Tuple

import torch

from . import decoder


class OutOfPages(RuntimeError):
    """The pool has too few free pages; nothing was changed."""


@dataclass
class Step:
    """What one forward pass needs for its new tokens, on the device."""

    positions: torch.Tensor   # int64 [T], rows of the rotary table
    slots: torch.Tensor       # int64 [T], where the new keys and values go
    page_table: torch.Tensor  # int32 [B, pages]
    q_starts: torch.Tensor    # int32 [B + 1]
    kv_lens: torch.Tensor     # int32 [B], the new tokens included
    max_q: int
    max_kv: int
    # the same of each sequence on the host (max_q and max_kv may be replaced by upper bounds)
    new_tokens: Optional[Tuple[int, ...]] = None
    lengths: Optional[Tuple[int, ...]] = None


class PagedCache:
    def __init__(self, layers: int, kv_heads: int, head_dim: int, pages: int, page_size: int = 16,
                 dtype: torch.dtype = torch.bfloat16, device="cuda"):
        if min(layers, kv_heads, head_dim, pages) < 1 or page_size < 16 or page_size & (page_size - 1):
            raise ValueError("layers, kv_heads, head_dim and pages must be positive, page_size a power of two from 16 up")
        self.page_size, self.pages = page_size, pages
        # (zeros: a page's unused tail is never read into a result, but a pool that starts finite
        # keeps dumps and comparisons simple)
        self.pool = torch.zeros((layers, 2, pages, kv_heads, page_size, head_dim), dtype=dtype, device=device)
        self._free = list(range(pages))  # a heap: the lowest free page is taken first
        self._refs = [0] * pages
        self._lists: Dict[int, List[int]] = {}
        self._lens: Dict[int, int] = {}
        self._next = 0

    # ---- what is there
    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, seq: int) -> int:
        return self._lens[seq]

    def pages_of(self, seq: int) -> List[int]:
        return list(self._lists[seq])

    def layer(self, i: int):
        """(k_cache, v_cache) of layer i, each [pages, kv_heads, page_size, head_dim]."""
        return self.pool[i, 0], self.pool[i, 1]

    # ---- sequences
    def new(self) -> int:
        seq, self._next = self._next, self._next + 1
        self._lists[seq], self._lens[seq] = [], 0
        return seq

    def fork(self, seq: int) -> int:
        """A sequence with the same contents; no page is copied yet."""
        pages, n = self._lists[seq], self._lens[seq]
        other = self.new()
        for p in pages:
            self._refs[p] += 1
        self._lists[other], self._lens[other] = list(pages), n
        return other

    def truncate(self, seq: int, length: int) -> None:
        """Drops the tokens from `length` on and frees the pages that held only them."""
        if not 0 <= length <= self._lens[seq]:
            raise ValueError(f"sequence {seq} holds {self._lens[seq]} tokens, cannot keep {length}")
        keep = -(-length // self.page_size)
        pages = self._lists[seq]
        self._drop(pages[keep:])
        del pages[keep:]
        self._lens[seq] = length

    def free(self, seq: int) -> None:
        self._drop(self._lists.pop(seq))
        del self._lens[seq]

    def _drop(self, pages: Sequence[int]) -> None:
        for p in pages:
            self._refs[p] -= 1
            if self._refs[p] == 0:
                heapq.heappush(self._free, p)

    def _take(self) -> int:
        p = heapq.heappop(self._free)
        self._refs[p] = 1
        return p

    # ---- a forward pass
    def step(self, seqs: Sequence[int], new_tokens: Sequence[int]) -> Step:
        """Room for new_tokens[i] more tokens of sequence seqs[i] (a sequence occurs once); returns
        the pass's index tensors.  A shared, partly filled last page is copied first (in all
        layers, one call).  Raises OutOfPages before anything changes."""
        if len(seqs) != len(new_tokens) or len(set(seqs)) != len(seqs) or not seqs:
            raise ValueError("expected distinct sequences and one token count for each")
        if min(new_tokens) < 0 or sum(new_tokens) == 0:
            raise ValueError("token counts must not be negative, and not all zero")
        ps = self.page_size
        need, seen = 0, {}
        for s, n in zip(seqs, new_tokens):
            have, pages = self._lens[s], self._lists[s]
            need += max(0, -(-(have + n) // ps) - len(pages))
            if n and have % ps:  # sharers of one page copy it but for the last that writes alone
                p = pages[-1]
                seen[p] = seen.get(p, 0) + 1
        need += sum(min(w, self._refs[p] - 1) for p, w in seen.items())
        if need > len(self._free):
            raise OutOfPages(f"{need} pages needed, {len(self._free)} free")
        src, dst = [], []
        positions, slots, starts, lens = [], [], [0], []
        for s, n in zip(seqs, new_tokens):
            have, pages = self._lens[s], self._lists[s]
            if n and have % ps and self._refs[pages[-1]] > 1:
                fresh = self._take()
                src.append(pages[-1])
                dst.append(fresh)
                self._drop([pages[-1]])
                pages[-1] = fresh
            while len(pages) * ps < have + n:
                pages.append(self._take())
            positions.extend(range(have, have + n))
            slots.extend(pages[i // ps] * ps + i % ps for i in range(have, have + n))
            self._lens[s] = have + n
            starts.append(starts[-1] + n)
            lens.append(have + n)
        if src:
            decoder.copy_pages(self.pool, src, dst)
        width = max(1, max(len(self._lists[s]) for s in seqs))
        table = [self._lists[s] + [-1] * (width - len(self._lists[s])) for s in seqs]
        dev = self.pool.device
        wide = torch.tensor([positions, slots], dtype=torch.int64).to(dev, non_blocking=True)
        flat = [x for row in table for x in row] + starts + lens
        small = torch.tensor(flat, dtype=torch.int32).to(dev, non_blocking=True)
        B = len(seqs)
        return Step(wide[0], wide[1], small[:B * width].view(B, width), small[B * width:B * width + B + 1],
                    small[B * width + B + 1:], max(new_tokens), max(lens), tuple(new_tokens), tuple(lens))

    # ---- the pool
    def compact(self) -> int:
        """Moves pages so that the used ones are the lowest; returns how many moved.  Slots and
        page tables from before are void."""
        used = [p for p in range(self.pages) if self._refs[p]]
        n = len(used)
        holes = [p for p in range(n) if not self._refs[p]]
        movers = [p for p in used if p >= n]
        if movers:
            decoder.copy_pages(self.pool, movers, holes)
        where = dict(zip(movers, holes))
        for pages in self._lists.values():
            pages[:] = [where.get(p, p) for p in pages]
        for a, b in where.items():
            self._refs[b], self._refs[a] = self._refs[a], 0
        self._free = list(range(n, self.pages))
        return len(movers)
