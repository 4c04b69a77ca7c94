"""A paged key-value cache for the decoder stack.

The cache of every layer is one pool of pages of ``page_size`` positions; a
sequence holds a list of pages, in order, that is the same in all layers.  So
sequences of any mix of lengths share the memory, they come and go one by one,
a prompt that several continuations share is held once, and with a window a
stream of any length stays within a bounded number of pages.

:class:`PageTables` is the bookkeeping (host data, no GPU): which pages are
free, how many sequences hold each, which copies a change needs.
:class:`PagedKVCache` adds the pools and runs those copies
(:func:`nki_moe_b200.ops.copy_pages`) on the current stream; use one cache from
one stream.

The reference keeps its caches in the runtime that it calls (one contiguous
region per sequence); nothing there corresponds to this module.
"""

from __future__ import annotations

import heapq

import torch

from . import ops

__all__ = ["PageTables", "PagedKVCache", "CacheFull"]


class CacheFull(RuntimeError):
    """No page is free for the positions asked for; nothing was changed."""


class _Sequence:
    def __init__(self, pages: list[int], length: int):
        self.pages, self.length = pages, length  # a page of -1 is not held (a window has passed it)


class PageTables:
    """Pages of ``num_pages`` in sequences of at most ``max_pages`` each.

    ``window``/``sinks``: what the attention sees (0: everything); pages that
    lie outside for every later position are given back by :meth:`trim`."""

    def __init__(self, num_pages: int, page_size: int, max_pages: int, window: int = 0, sinks: int = 0):
        if page_size not in ops._PAGE_SIZES:
            raise ValueError(f"page size {page_size} (one of {ops._PAGE_SIZES})")
        if num_pages <= 0 or max_pages <= 0 or window < 0 or sinks < 0:
            raise ValueError("num_pages and max_pages must be positive, window and sinks not negative")
        self.num_pages, self.page_size, self.max_pages = num_pages, page_size, max_pages
        self.window, self.sinks = window, sinks
        self._free = list(range(num_pages))  # a heap: the lowest ids are used first
        self._refs = [0] * num_pages
        self._seqs: dict[int, _Sequence] = {}
        self._next = 0

    # ------------------------------------------------------------ reading
    @property
    def free_pages(self) -> int:
        return len(self._free)

    def __contains__(self, seq: int) -> bool:
        return seq in self._seqs

    def _seq(self, seq: int) -> _Sequence:
        try:
            return self._seqs[seq]
        except KeyError:
            raise ValueError(f"no sequence {seq}") from None

    def length(self, seq: int) -> int:
        return self._seq(seq).length

    def pages(self, seq: int) -> list[int]:
        return list(self._seq(seq).pages)

    # ------------------------------------------------------------ sequences
    def add(self) -> int:
        """A new, empty sequence."""
        seq, self._next = self._next, self._next + 1
        self._seqs[seq] = _Sequence([], 0)
        return seq

    def fork(self, seq: int) -> int:
        """A new sequence that goes on from where ``seq`` stands.  The two
        share their pages; the one that is written first gets its own copy of
        the last one then (:meth:`extend`)."""
        s = self._seq(seq)
        for p in s.pages:
            if p >= 0:
                self._refs[p] += 1
        new = self.add()
        self._seqs[new] = _Sequence(list(s.pages), s.length)
        return new

    def _drop(self, page: int) -> None:
        if page >= 0:
            self._refs[page] -= 1
            if self._refs[page] == 0:
                heapq.heappush(self._free, page)

    def free(self, seq: int) -> None:
        """Ends a sequence; the pages that it held alone are free again."""
        for p in self._seq(seq).pages:
            self._drop(p)
        del self._seqs[seq]

    def extend(self, seqs, counts) -> list[tuple[int, int]]:
        """Makes room for ``counts[i]`` more positions in ``seqs[i]`` (each
        sequence once) and counts them in its length.  Returns the copies
        (source page, new page) that make the pages to be written private.
        Raises :class:`CacheFull`, with nothing changed, if pages are short."""
        seqs, counts = list(seqs), list(counts)
        if len(seqs) != len(counts) or len(set(seqs)) != len(seqs) or any(c < 0 for c in counts):
            raise ValueError("one count, not negative, for each of different sequences")
        need = 0
        shared = []
        copied: dict[int, int] = {}  # how many of this call's sequences copy a page
        for q, c in zip(seqs, counts):
            s = self._seq(q)
            total = -(-(s.length + c) // self.page_size)
            if total > self.max_pages:
                raise ValueError(f"sequence {q}: {s.length + c} positions, the page table takes "
                                 f"{self.max_pages * self.page_size}")
            own = False
            if c and s.length % self.page_size:
                page = s.pages[-1]
                # the last of the sequences that share it may keep it
                own = page < 0 or self._refs[page] - copied.get(page, 0) <= 1
                if not own:
                    copied[page] = copied.get(page, 0) + 1
            shared.append(bool(c) and s.length % self.page_size != 0 and not own)
            need += total - len(s.pages) + shared[-1]
        if need > len(self._free):
            raise CacheFull(f"{need} pages are needed, {len(self._free)} are free")
        copies = []
        for q, c, copy in zip(seqs, counts, shared):
            s = self._seqs[q]
            if copy:
                old, new = s.pages[-1], self._take()
                copies.append((old, new))
                self._drop(old)
                s.pages[-1] = new
            s.length += c
            while len(s.pages) * self.page_size < s.length:
                s.pages.append(self._take())
        return copies

    def take_back(self, seqs, lengths) -> None:
        """Puts ``seqs[i]`` back to ``lengths[i]`` positions, as it had before an
        :meth:`extend` whose positions were not written after all.  The pages
        behind are given back; one that was made private stays so."""
        seqs, lengths = list(seqs), list(lengths)
        if len(seqs) != len(lengths) or any(not 0 <= n <= self.length(q) for q, n in zip(seqs, lengths)):
            raise ValueError("one length, no larger than the sequence's, for each sequence")
        for q, n in zip(seqs, lengths):
            s = self._seqs[q]
            while len(s.pages) > -(-n // self.page_size):
                self._drop(s.pages.pop())
            s.length = n

    def _take(self) -> int:
        page = heapq.heappop(self._free)
        self._refs[page] = 1
        return page

    def trim(self, seq: int) -> int:
        """Gives back the pages of ``seq`` that no later position sees (with a
        window: those before it and behind the first ``sinks`` positions).
        Returns how many."""
        s = self._seq(seq)
        if not self.window:
            return 0
        first = s.length - self.window + 1  # the next position, s.length, sees from here on
        dropped = 0
        for i in range(-(-self.sinks // self.page_size), min(len(s.pages), max(0, first) // self.page_size)):
            if s.pages[i] >= 0:
                self._drop(s.pages[i])
                s.pages[i] = -1
                dropped += 1
        return dropped

    def compact(self) -> list[tuple[int, int]]:
        """Moves the pages in use to the front of the pool; returns the copies
        (from, to), of which no page is both.  Sequences keep their ids."""
        used = [p for p in range(self.num_pages) if self._refs[p]]
        n = len(used)
        moves = dict(zip([p for p in used if p >= n], [p for p in range(n) if not self._refs[p]]))
        for s in self._seqs.values():
            s.pages = [moves.get(p, p) for p in s.pages]
        for a, b in moves.items():
            self._refs[b], self._refs[a] = self._refs[a], 0
        self._free = list(range(n, self.num_pages))
        return sorted(moves.items())

    def table(self, seqs) -> torch.Tensor:
        """The page table of ``seqs`` in that order: int32 ``[len(seqs),
        max_pages]`` on the CPU, -1 where no page is held."""
        t = torch.full((len(seqs), self.max_pages), -1, dtype=torch.int32)
        for i, q in enumerate(seqs):
            pages = self._seq(q).pages
            if pages:
                t[i, :len(pages)] = torch.tensor(pages, dtype=torch.int32)
        return t


class PagedKVCache(PageTables):
    """:class:`PageTables` with the pools of ``num_layers`` layers on a GPU:
    ``pool [num_layers, 2, num_pages, n_kv_heads, page_size, 128]`` bf16, keys
    and values."""

    def __init__(self, num_layers: int, n_kv_heads: int, num_pages: int, page_size: int = 64, max_seq: int = 4096,
                 window: int = 0, sinks: int = 0, device="cuda"):
        super().__init__(num_pages, page_size, -(-max_seq // page_size) if page_size > 0 else 1, window, sinks)
        self.device = torch.device(device)
        self.pool = torch.empty(num_layers, 2, num_pages, n_kv_heads, page_size, 128, dtype=torch.bfloat16,
                                device=self.device)

    def layer(self, i: int) -> tuple[torch.Tensor, torch.Tensor]:
        """Layer ``i``'s ``k_pages``, ``v_pages``."""
        return self.pool[i, 0], self.pool[i, 1]

    def _copy(self, copies: list[tuple[int, int]]) -> None:
        if copies:
            ops.copy_pages(self.pool, [a for a, _ in copies], [b for _, b in copies])

    def extend(self, seqs, counts) -> list[tuple[int, int]]:
        copies = super().extend(seqs, counts)
        self._copy(copies)
        return copies

    def compact(self) -> list[tuple[int, int]]:
        copies = super().compact()
        self._copy(copies)
        return copies
