"""Ownership of a paged KV cache: which page of the pool belongs to which sequences.

The pool of all layers is one tensor [2 * n_layers, n_pages, page, Hkv, D] (keys of layer i in row 2 i, values in row 2 i + 1);
a page id means the same page in every row, so forks and compaction are one ``copy_pages`` launch for the whole model. The
bookkeeping (free list, reference counts, page lists) lives on the host; the device sees block tables made by ``table``.

    cache = PagedCache(n_layers, n_pages, page_size, n_kv_heads, head_dim)
    s = cache.add()                     # an empty sequence
    cache.reserve([s], [len(prompt)])   # room for its next tokens; append / attend with cache.table([s]), cache.length(s)
    a, b = cache.fork(s, 2)             # two continuations that share every page, the last one until it is written to
    cache.release_behind(s, 1024, 4)    # give back what a window of 1024 and 4 first tokens do not reach
    cache.free(s)

Work on the pool is queued on the current stream: use one stream for a cache, or order the streams.
"""
from __future__ import annotations

from typing import Dict, List, Optional, Sequence, Tuple

import torch

from .ops.paged import PAGE_SIZES, copy_pages


class CacheFull(RuntimeError):
    """A reservation needs more pages than are free. Nothing was changed."""


class PagedCache:
    def __init__(self, n_layers: int, n_pages: int, page_size: int, n_kv_heads: int, head_dim: int,
                 dtype: torch.dtype = torch.bfloat16, device="cuda"):
        if page_size not in PAGE_SIZES:
            raise ValueError(f"page size must be one of {PAGE_SIZES}, got {page_size}")
        if min(n_layers, n_pages, n_kv_heads, head_dim) < 1:
            raise ValueError("a cache needs at least one layer, page, head and channel")
        self.n_layers, self.page_size = n_layers, page_size
        self.pool = torch.zeros(2 * n_layers, n_pages, page_size, n_kv_heads, head_dim, dtype=dtype, device=device)
        self._free: List[int] = list(range(n_pages - 1, -1, -1))  # taken from the end: low ids first
        self._refs = [0] * n_pages
        self._pages: Dict[int, List[int]] = {}  # page of every block of positions; -1: given back
        self._len: Dict[int, int] = {}
        self._next = 0

    # ---- the pool
    @property
    def n_pages(self) -> int:
        return self.pool.shape[1]

    @property
    def n_free(self) -> int:
        return len(self._free)

    def layer(self, i: int) -> Tuple[torch.Tensor, torch.Tensor]:
        """(k_pages, v_pages) of layer i, [n_pages, page, Hkv, D] views of the pool."""
        return self.pool[2 * i], self.pool[2 * i + 1]

    # ---- sequences
    def add(self) -> int:
        s, self._next = self._next, self._next + 1
        self._pages[s], self._len[s] = [], 0
        return s

    def length(self, seq: int) -> int:
        return self._len[seq]

    def pages(self, seq: int) -> List[int]:
        return list(self._pages[seq])

    def _take(self) -> int:
        p = self._free.pop()
        self._refs[p] = 1
        return p

    def _drop(self, page: int) -> None:
        self._refs[page] -= 1
        if self._refs[page] == 0:
            self._free.append(page)

    def reserve(self, seqs: Sequence[int], n_new: Sequence[int]) -> bool:
        """Lengthens every sequence by its number of new tokens and finds pages for them; a shared page that one of them
        would write into is copied first. Returns whether any page list changed. Raises CacheFull, with nothing changed,
        if the pool has too few free pages."""
        if len(seqs) != len(n_new) or len(set(seqs)) != len(seqs):
            raise ValueError("reserve takes one number of tokens for each of several different sequences")
        if any(n < 0 for n in n_new):
            raise ValueError("a sequence cannot grow by a negative number of tokens")
        P = self.page_size
        left = {}  # references a page would have left as copies are made for its writers, one after the other
        need, plan = 0, []
        for s, n in zip(seqs, n_new):
            pages, length = self._pages[s], self._len[s]
            fresh = (length + n + P - 1) // P - len(pages)
            copy = False
            if n > 0 and length % P:
                last = pages[-1]
                r = left.get(last, self._refs[last])
                copy = r > 1
                left[last] = r - 1 if copy else r
            need += fresh + copy
            plan.append((s, n, fresh, copy))
        if need > len(self._free):
            raise CacheFull(f"{need} pages needed, {len(self._free)} of {self.n_pages} free")
        src, dst = [], []
        for s, n, fresh, copy in plan:
            pages = self._pages[s]
            if copy:
                src.append(pages[-1])
                self._refs[pages[-1]] -= 1  # never the last reference: another sequence keeps the page
                pages[-1] = self._take()
                dst.append(pages[-1])
            pages.extend(self._take() for _ in range(fresh))
            self._len[s] += n
        if src:
            copy_pages(self.pool, torch.tensor(src, dtype=torch.int32), torch.tensor(dst, dtype=torch.int32))
        return need > 0

    def fork(self, seq: int, n: int = 1) -> List[int]:
        """n new sequences with the contents of ``seq``. Nothing is copied until one of them grows."""
        out = []
        for _ in range(n):
            s = self.add()
            self._pages[s], self._len[s] = list(self._pages[seq]), self._len[seq]
            for p in self._pages[s]:
                if p >= 0:
                    self._refs[p] += 1
            out.append(s)
        return out

    def free(self, seq: int) -> None:
        for p in self._pages.pop(seq):
            if p >= 0:
                self._drop(p)
        del self._len[seq]

    def release_behind(self, seq: int, window: int, sinks: int = 0) -> bool:
        """Gives back the pages that no later token of ``seq`` sees with this window and these first tokens. Returns
        whether there were any."""
        if window <= 0:
            return False
        pages, P = self._pages[seq], self.page_size
        first = max(0, self._len[seq] - window + 1)  # first key inside the window of the next token
        changed = False
        for c in range((max(sinks, 0) + P - 1) // P, first // P):
            if pages[c] >= 0:
                self._drop(pages[c])
                pages[c] = -1
                changed = True
        return changed

    def compact(self) -> int:
        """Moves the pages in use to the lowest ids, in one launch, and returns how many there are. Block tables made
        before are stale."""
        used = [p for p, r in enumerate(self._refs) if r > 0]
        n = len(used)
        holes = [p for p in range(n) if self._refs[p] == 0]
        src = used[n - len(holes):]  # as many pages in use lie at or above n as there are holes below
        if src:
            copy_pages(self.pool, torch.tensor(src, dtype=torch.int32), torch.tensor(holes, dtype=torch.int32))
            to = dict(zip(src, holes))
            for pages in self._pages.values():
                pages[:] = [to.get(p, p) for p in pages]
            for a, b in to.items():
                self._refs[b], self._refs[a] = self._refs[a], 0
        self._free = list(range(self.n_pages - 1, n - 1, -1))
        return n

    def resize(self, n_pages: int) -> None:
        """A pool of another number of pages with the same contents (compacted first if pages would be lost). The views
        that ``layer`` returned before belong to the old pool."""
        used = sum(r > 0 for r in self._refs)
        if n_pages < max(used, 1):
            raise CacheFull(f"{used} pages are in use, {n_pages} wanted")
        if n_pages < self.n_pages:
            self.compact()
        keep = min(n_pages, self.n_pages)
        pool = self.pool.new_zeros(self.pool.shape[0], n_pages, *self.pool.shape[2:])
        pool[:, :keep] = self.pool[:, :keep]
        self.pool = pool
        self._refs = self._refs[:keep] + [0] * (n_pages - keep)
        self._free = [p for p in range(n_pages - 1, -1, -1) if self._refs[p] == 0]

    def table(self, seqs: Sequence[int], cols: Optional[int] = None) -> torch.Tensor:
        """Block table [len(seqs), cols] (int32, host) of the pages of these sequences, -1 where there is none."""
        width = max((len(self._pages[s]) for s in seqs), default=0)
        cols = max(width, 1) if cols is None else cols
        if width > cols:
            raise ValueError(f"a sequence has {width} pages, the table {cols} columns")
        t = torch.full((len(seqs), cols), -1, dtype=torch.int32)
        for i, s in enumerate(seqs):
            p = self._pages[s]
            t[i, :len(p)] = torch.tensor(p, dtype=torch.int32)
        return t
