"""A paged key / value cache: one pool of pages for all layers, sequences as lists of pages.

``PagedCache`` keeps the books on the host (which page belongs to whom, how often it is shared) and
touches the device only where pages are copied: a fork shares its pages and copies the last one,
if it is partly filled, when one of the two first writes to it; ``compact`` moves pages down.
``step`` turns "these sequences get so many new tokens" into the index tensors that
``rope_append`` and ``paged_attention`` take; ``ahead`` reserves pages for many steps of one token, whose
index tensors then come from the GPU alone (``decoder.plan_step``), so that a step can be captured
in a graph.  ``evict`` gives back the pages that a window with sinks has left behind.
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
        self._lists: Dict[int, List[int]] = {}  # -1: an evicted page
        self._lens: Dict[int, int] = {}
        self._least: Dict[int, int] = {}  # the length that an evicted sequence cannot be truncated below
        self._lent: Dict[int, "Ahead"] = {}  # sequences whose steps an Ahead plans
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
        self._keeps(seq)
        pages, n = self._lists[seq], self._lens[seq]
        other = self.new()
        for p in pages:
            if p >= 0:
                self._refs[p] += 1
        self._lists[other], self._lens[other] = list(pages), n
        if seq in self._least:
            self._least[other] = self._least[seq]
        return other

    def truncate(self, seq: int, length: int) -> None:
        """Drops the tokens from `length` on and frees the pages that held only them."""
        self._keeps(seq)
        if not 0 <= length <= self._lens[seq]:
            raise ValueError(f"sequence {seq} holds {self._lens[seq]} tokens, cannot keep {length}")
        if length < self._least.get(seq, 0):
            raise ValueError(f"sequence {seq} has lost pages that its tokens before {self._least[seq]} would see, cannot keep {length}")
        keep = -(-length // self.page_size)
        pages = self._lists[seq]
        self._drop(pages[keep:])
        del pages[keep:]
        self._lens[seq] = length

    def free(self, seq: int) -> None:
        self._keeps(seq)
        self._drop(self._lists.pop(seq))
        del self._lens[seq]
        self._least.pop(seq, None)

    def evict(self, seq: int, window: int, sinks: int = 0) -> int:
        """Gives back the pages that no further token of the sequence sees, where each sees the last
        ``window`` positions and the first ``sinks`` (``paged_attention``'s window and sinks); returns how many.
        Their places in the page list say -1; the sequence can no longer be truncated below its present length."""
        self._keeps(seq)
        if window < 1 or sinks < 0:
            raise ValueError(f"a window must be positive and sinks not negative, got {window} and {sinks}")
        ps, pages, n = self.page_size, self._lists[seq], self._lens[seq]
        gone = [i for i in range(-(-sinks // ps), max(0, n + 1 - window) // ps) if pages[i] >= 0]
        self._drop([pages[i] for i in gone])
        for i in gone:
            pages[i] = -1
        if gone:
            self._least[seq] = n
        return len(gone)

    def _keeps(self, seq: int) -> None:
        if seq in self._lent:
            raise ValueError(f"sequence {seq} has steps planned ahead; close them first")

    def _drop(self, pages: Sequence[int]) -> None:
        for p in pages:
            if p < 0:
                continue
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
        if min(new_tokens, default=0) < 0 or sum(new_tokens) == 0:
            raise ValueError("token counts must not be negative, and not all zero")
        ps, B = self.page_size, len(seqs)
        self._room(seqs, new_tokens)
        self._unshare([s for s, n in zip(seqs, new_tokens) if n])
        had, lens = [self._lens[s] for s in seqs], []
        for s, n in zip(seqs, new_tokens):
            pages = self._lists[s]
            while len(pages) * ps < self._lens[s] + n:
                pages.append(self._take())
            self._lens[s] += n
            lens.append(self._lens[s])
        table, width = self._table(seqs, 1)
        dev = self.pool.device
        if dev.type == "cuda":  # the host names the pages, the GPU places the tokens
            small = torch.tensor(table + had + list(new_tokens), dtype=torch.int32).to(dev, non_blocking=True)
            view = small[:B * width].view(B, width)
            positions, slots, starts, kv_lens, _ = decoder.plan_step(
                view, small[B * width:B * width + B], small[B * width + B:], page_size=ps, max_tokens=sum(new_tokens))
        else:
            at = [i for n, h in zip(new_tokens, had) for i in range(h, h + n)]
            owner = [s for s, n in zip(seqs, new_tokens) for _ in range(n)]
            positions = torch.tensor(at, dtype=torch.int64)
            slots = torch.tensor([self._lists[s][i // ps] * ps + i % ps for s, i in zip(owner, at)], dtype=torch.int64)
            starts = torch.tensor([0] + list(new_tokens)).cumsum(0).int()
            kv_lens, view = torch.tensor(lens, dtype=torch.int32), torch.tensor(table, dtype=torch.int32).view(B, width)
        return Step(positions, slots, view, starts, kv_lens, max(new_tokens), max(lens), tuple(new_tokens), tuple(lens))

    def ahead(self, seqs: Sequence[int], steps: int) -> "Ahead":
        """Room for ``steps`` steps of one token more of each sequence (a sequence occurs once), planned on
        the GPU one by one.  Until the returned ``Ahead`` is closed, these sequences belong to it."""
        return Ahead(self, seqs, steps)

    def ahead_of(self, seq: int) -> Optional["Ahead"]:
        """The open ``Ahead`` that plans the sequence's steps, to be closed by who has lost it; None if there is none."""
        return self._lent.get(seq)

    def _room(self, seqs: Sequence[int], new_tokens: Sequence[int]) -> int:
        """Pages that the tokens need beyond those there, without copies of shared ones."""
        if len(seqs) != len(new_tokens) or len(set(seqs)) != len(seqs) or not seqs:
            raise ValueError("expected distinct sequences and one token count for each")
        ps, need, seen = self.page_size, 0, {}
        for s, n in zip(seqs, new_tokens):
            self._keeps(s)
            have, pages = self._lens[s], self._lists[s]
            need += max(0, -(-(have + n) // ps) - len(pages))
            if n and have % ps:  # sharers of one page copy it but for the last that writes alone
                p = pages[-1]
                seen[p] = seen.get(p, 0) + 1
        copies = sum(min(w, self._refs[p] - 1) for p, w in seen.items())
        if need + copies > len(self._free):
            raise OutOfPages(f"{need + copies} pages needed, {len(self._free)} free")
        return need

    def _unshare(self, seqs: Sequence[int]) -> None:
        """Copies the last pages, where partly filled, that the sequences share."""
        src, dst = [], []
        for s in seqs:
            pages = self._lists[s]
            if self._lens[s] % self.page_size and self._refs[pages[-1]] > 1:
                fresh = self._take()
                src.append(pages[-1])
                dst.append(fresh)
                self._drop([pages[-1]])
                pages[-1] = fresh
        if src:
            decoder.copy_pages(self.pool, src, dst)

    def _table(self, seqs: Sequence[int], width: int):
        """The page lists one after the other, each filled up with -1 to the longest (or width), and that."""
        width = max(width, max(len(self._lists[s]) for s in seqs))
        return [p for s in seqs for p in self._lists[s] + [-1] * (width - len(self._lists[s]))], width

    # ---- the pool
    def compact(self) -> int:
        """Moves pages so that the used ones are the lowest; returns how many moved.  Slots and
        page tables from before are void."""
        for seq in self._lent:
            self._keeps(seq)
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


class Ahead:
    """Steps of one token for each of some sequences, with their pages reserved and every step's index
    tensors made on the GPU from the lengths of the step before: ``next`` uploads nothing and waits for nothing,
    and may be captured in a graph and replayed, up to ``steps`` times in all; a replay beyond them has no tokens, and
    ``device_error()`` tells.  ``close`` tells the cache how many steps ran; a captured step must not be replayed after
    it (its pages may be another sequence's by then).  The cache holds it until then (``ahead_of``): one that a program drops
    may still be captured in its graphs."""

    def __init__(self, cache: PagedCache, seqs: Sequence[int], steps: int):
        if steps < 1:
            raise ValueError(f"at least one step, got {steps}")
        self.cache, self.seqs, self.steps = cache, list(seqs), steps
        self._called = 0  # steps that `next` itself ran
        need = cache._room(self.seqs, [steps] * len(self.seqs))
        cache._unshare(self.seqs)
        self._free = [cache._take() for _ in range(need)]
        B, ps, dev = len(self.seqs), cache.page_size, cache.pool.device
        had = [cache._lens[s] for s in self.seqs]
        self.max_kv = max(had) + steps
        try:
            table, width = cache._table(self.seqs, -(-self.max_kv // ps))
            small = torch.tensor(table + had + [1] * B + self._free + [0], dtype=torch.int32).to(dev, non_blocking=True)
            self._table = small[:B * width].view(B, width)
            self._lengths, self._ones, rest = small[B * width:B * width + B], small[B * width + B:B * width + 2 * B], small[B * width + 2 * B:]
            self._pages, taken = rest[:need], rest[need:]
            wide = torch.zeros(2 * B, dtype=torch.int64, device=dev)
            self._out = (wide[:B], wide[B:], torch.zeros(B + 1, dtype=torch.int32, device=dev), self._lengths, taken)
        except BaseException:  # (no memory on the device)
            cache._drop(self._free)
            raise
        cache._lent.update(dict.fromkeys(self.seqs, self))
        self._open = True

    def next(self) -> Step:
        """The next step; its tensors are those of the step before, written again.  More calls than steps raise
        ValueError.  After ``close`` a step has no tokens (slots -1), whatever became of its pages, and ``device_error()`` tells."""
        B, ps = len(self.seqs), self.cache.page_size
        if not self._open:  # (counts below 0: no room)
            positions, slots, starts, lens, _ = decoder.plan_step(
                self._table, self._lengths, torch.full_like(self._ones, -1), page_size=ps, max_tokens=B)
            return Step(positions, slots, self._table, starts, lens, 1, self.max_kv)
        if not torch.cuda.is_current_stream_capturing():
            if self._called == self.steps:
                raise ValueError(f"all {self.steps} reserved steps have run")
            self._called += 1
        positions, slots, starts, lens, _ = decoder.plan_step(
            self._table, self._lengths, self._ones, page_size=ps, max_tokens=B, max_kv=self.max_kv, free_pages=self._pages,
            taken=self._out[4], out=self._out)
        return Step(positions, slots, self._table, starts, lens, 1, self.max_kv)

    def close(self, done: int) -> None:
        """Enters ``done`` steps in the cache's books and gives back the pages that they did not need."""
        if not self._open:
            return
        if not 0 <= done <= self.steps:
            raise ValueError(f"{self.steps} steps were reserved, {done} cannot have run")
        c = self.cache
        for s in self.seqs:
            del c._lent[s]
        self._open = False
        at = 0
        for _ in range(done):  # pages were taken in the order of the steps, in each of the sequences
            for s in self.seqs:
                if c._lens[s] % c.page_size == 0:
                    c._lists[s].append(self._free[at])
                    at += 1
                c._lens[s] += 1
        c._drop(self._free[at:])
