"""The pages of a 4-bit cache on the host: which are free, whose they are, and what has to be copied.

``KV4Cache`` holds the cache tensor of one layer (or any number of layers that share their page numbers, one tensor each) and the
page lists of the sequences in it. Pages are counted: a fork shares its parent's full pages and copies the one that both would go on
writing to; a page is free once the last sequence that holds it is gone. ``compact`` moves the pages in use to the front, so that
what lies behind them can be given back. Pages are copied by ``ops.copy_pages`` on the current stream. Slots and tables are built from
Python lists and copied from ordinary host memory, which may hold up the host until the copy is made: for 64 sequences of 512 to 8192
tokens the lists take 0.4 ms (``extend`` of each by one) and 0.8 ms (``tables``), once for all layers of a step.
"""
from __future__ import annotations

from typing import Dict, List, Sequence, Tuple

import torch

from . import ops


class KV4Cache:
    def __init__(self, pages: int, kv_heads: int, head_dim: int, page_size: int = 64, layers: int = 1, device="cuda"):
        if pages < 1 or kv_heads < 1 or layers < 1 or head_dim not in (64, 128, 256) or page_size < 16 or page_size % 16:
            raise ValueError("KV4Cache: pages of a multiple of 16 tokens, head_dim 64, 128 or 256")
        self.page_size = page_size
        self.layers = [torch.zeros(pages, kv_heads, page_size // 16, 18 * head_dim, dtype=torch.uint8, device=device) for _ in range(layers)]
        self._holders = [0] * pages
        self._free = list(range(pages - 1, -1, -1))  # taken from the end: lowest numbers first
        self._pages: Dict[int, List[int]] = {}
        self._length: Dict[int, int] = {}
        self._next = 0

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, seq: int) -> int:
        return self._length[seq]

    def pages(self, seq: int) -> Tuple[int, ...]:
        return tuple(self._pages[seq])

    def new(self) -> int:
        """A sequence without tokens."""
        seq, self._next = self._next, self._next + 1
        self._pages[seq], self._length[seq] = [], 0
        return seq

    def _take(self, count: int) -> List[int]:
        if count > len(self._free):
            raise MemoryError(f"KV4Cache: {count} pages asked for, {len(self._free)} free")
        taken = [self._free.pop() for _ in range(count)]
        for p in taken:
            self._holders[p] = 1
        return taken

    def _drop(self, pages: Sequence[int]) -> None:
        for p in pages:
            self._holders[p] -= 1
            if self._holders[p] == 0:
                self._free.append(p)

    def _copy(self, src: List[int], dst: List[int]) -> None:
        if src:
            for layer in self.layers:
                ops.copy_pages(layer, src, dst)

    def extend(self, seq: int, tokens: int) -> torch.Tensor:
        """Room for `tokens` more tokens of a sequence: their slots (int64, on the cache's device), for kv4_append."""
        if tokens < 0:
            raise ValueError("KV4Cache: a negative number of tokens")
        pages, n, size = self._pages[seq], self._length[seq], self.page_size
        held = len(pages)
        pages += self._take(-(-(n + tokens) // size) - held)
        try:
            slots = torch.tensor([pages[i // size] * size + i % size for i in range(n, n + tokens)], dtype=torch.int64)
            slots = slots.to(self.layers[0].device, non_blocking=True)
        except BaseException:
            self._drop(pages[held:][::-1])
            del pages[held:]
            raise
        self._length[seq] = n + tokens
        return slots

    def fork(self, seq: int) -> int:
        """Another sequence with the same tokens. Full pages are shared; the last one, if it is not full, is copied."""
        pages, n = self._pages[seq], self._length[seq]
        full = n // self.page_size
        own = self._take(len(pages) - full)  # (before anything is changed)
        try:
            self._copy(pages[full:], own)
        except BaseException:
            self._drop(own[::-1])
            raise
        for p in pages[:full]:
            self._holders[p] += 1
        twin = self.new()
        self._pages[twin], self._length[twin] = pages[:full] + own, n
        return twin

    def free(self, seq: int) -> None:
        """Ends a sequence. Its pages may go to the next one at once: kernels that read them are in front on the stream, or waited for."""
        self._drop(self._pages.pop(seq))
        del self._length[seq]

    def compact(self) -> int:
        """Moves the pages in use to the front and returns how many they are. Slots and tables handed out before are stale."""
        used = [p for p, holders in enumerate(self._holders) if holders]
        gaps = [p for p, holders in enumerate(self._holders[:len(used)]) if not holders]
        src = [p for p in used if p >= len(used)]  # as many as there are gaps, and none of them one
        self._copy(src, gaps)
        moved = dict(zip(src, gaps))
        for a, b in moved.items():
            self._holders[b], self._holders[a] = self._holders[a], 0
        for pages in self._pages.values():
            pages[:] = [moved.get(p, p) for p in pages]
        self._free = list(range(len(self._holders) - 1, len(used) - 1, -1))
        return len(used)

    def tables(self, seqs: Sequence[int]) -> Tuple[torch.Tensor, torch.Tensor]:
        """(page_table, kv_lens) of these sequences for kv4_attention, on the cache's device. Places behind a list hold -1."""
        rows = [self._pages[s] for s in seqs]
        wide = max((len(r) for r in rows), default=0)
        table = torch.tensor([r + [-1] * (wide - len(r)) for r in rows], dtype=torch.int64).reshape(len(rows), wide)
        lens = torch.tensor([self._length[s] for s in seqs], dtype=torch.int64)
        device = self.layers[0].device
        return table.to(device, non_blocking=True), lens.to(device, non_blocking=True)
