"""Paged FP8 KV cache: sequences hold lists of fixed-size pages instead of one
max_seq row each, so that memory follows their lengths and forked sequences
share the pages of their common prefix.

``PageAllocator`` is the bookkeeping alone (host memory, no device): which
pages a sequence has, how many sequences share a page, and the page copies
and block-table cells that each operation calls for.  ``PagedKVCache`` holds
the pages of all layers and the block table on the GPU and carries those plans
out with ``ops.kv_copy_pages`` / ``ops.kv_table_set`` on the current stream.
The reference keeps one contiguous cache per request
(api_server.py:58-150) and has no counterpart."""
from __future__ import annotations

from dataclasses import dataclass, field
from typing import Optional, Sequence

import torch

from . import ops


class OutOfPages(RuntimeError):
    """The pool has too few free pages for a request; nothing was changed."""


@dataclass
class Plan:
    """Page copies (src[i] -> dst[i]) and block-table cells
    (table[rows[i], cols[i]] = values[i]) that carry out one operation.  The
    copied pages are never also written by the same plan."""
    src: list = field(default_factory=list)
    dst: list = field(default_factory=list)
    rows: list = field(default_factory=list)
    cols: list = field(default_factory=list)
    values: list = field(default_factory=list)

    def cell(self, row: int, col: int, page: int) -> None:
        self.rows.append(row)
        self.cols.append(col)
        self.values.append(page)


class PageAllocator:
    """Pages of ``seqs`` sequences out of a pool of ``n_pages`` pages of ``page``
    positions; a sequence holds at most ``max_blocks`` pages.  Pages are handed
    out lowest id first.  Every operation returns the Plan that has to run
    before the pages are used."""

    def __init__(self, n_pages: int, page: int, seqs: int, max_blocks: int):
        if n_pages < 1 or page < 16 or page % 16 or seqs < 1 or max_blocks < 1:
            raise ValueError(f"bad pool: {n_pages} pages of {page} positions (a multiple of 16), "
                             f"{seqs} sequences of {max_blocks} blocks")
        self.n_pages, self.page, self.seqs, self.max_blocks = int(n_pages), int(page), int(seqs), int(max_blocks)
        self.free_pages = list(range(n_pages - 1, -1, -1))      # a stack; kept with the lowest id on top
        self.refs = [0] * n_pages
        self.blocks: list = [[] for _ in range(seqs)]
        self.lengths = [0] * seqs

    @property
    def free_count(self) -> int:
        return len(self.free_pages)

    def _seq(self, s: int) -> int:
        if not 0 <= s < self.seqs:
            raise ValueError(f"sequence {s} outside [0, {self.seqs})")
        return s

    def _take(self) -> int:
        p = self.free_pages.pop()
        self.refs[p] = 1
        return p

    def _drop(self, p: int) -> None:
        self.refs[p] -= 1
        if self.refs[p] == 0:
            self.free_pages.append(p)

    def _sort_free(self) -> None:
        self.free_pages.sort(reverse=True)

    def extend(self, counts: dict) -> Plan:
        """Makes room for counts[s] more positions of every sequence s and
        advances its length.  A page that is shared and will be written (the
        partly filled last page of a fork) is replaced by a copy.  All or
        nothing: OutOfPages changes nothing."""
        need, refs = 0, {}
        for s, n in counts.items():
            self._seq(s)
            if n < 0:
                raise ValueError(f"sequence {s}: cannot extend by {n}")
            have, end = self.lengths[s], self.lengths[s] + n
            blocks = -(-end // self.page)
            if blocks > self.max_blocks:
                raise ValueError(f"sequence {s}: {end} positions exceed {self.max_blocks} pages of {self.page}")
            need += max(0, blocks - len(self.blocks[s]))
            if n and have % self.page:
                p = self.blocks[s][have // self.page]
                r = refs.setdefault(p, self.refs[p])
                if r > 1:
                    need += 1
                    refs[p] = r - 1
        if need > len(self.free_pages):
            raise OutOfPages(f"{need} pages needed, {len(self.free_pages)} free")
        plan = Plan()
        for s, n in counts.items():
            have, end, mine = self.lengths[s], self.lengths[s] + n, self.blocks[s]
            if n and have % self.page:
                i = have // self.page
                old = mine[i]
                if self.refs[old] > 1:
                    mine[i] = self._take()
                    plan.src.append(old)
                    plan.dst.append(mine[i])
                    plan.cell(s, i, mine[i])
                    self.refs[old] -= 1
            while len(mine) * self.page < end:
                mine.append(self._take())
                plan.cell(s, len(mine) - 1, mine[-1])
            self.lengths[s] = end
        return plan

    def check_writable(self, seq: int, end: int, start: int = 0) -> None:
        """ValueError unless the sequence holds positions [start, end) on pages that no other one shares."""
        if self.lengths[self._seq(seq)] < end:
            raise ValueError(f"sequence {seq} holds {self.lengths[seq]} positions, not {end}")
        shared = [p for p in self.blocks[seq][start // self.page:-(-end // self.page)] if self.refs[p] > 1]
        if shared:
            raise ValueError(f"sequence {seq} shares pages {shared[:4]} with another one")

    def fork(self, parent: int, child: int, length: Optional[int] = None) -> Plan:
        """The empty sequence ``child`` gets the first ``length`` positions of
        ``parent`` (default: all, also those reserved and not written yet), by
        sharing their pages."""
        self._seq(parent)
        self._seq(child)
        length = self.lengths[parent] if length is None else int(length)
        if not 0 <= length <= self.lengths[parent]:
            raise ValueError(f"sequence {parent} has {self.lengths[parent]} positions, not {length}")
        if self.blocks[child]:
            raise ValueError(f"sequence {child} is not empty")
        plan = Plan()
        for i in range(-(-length // self.page)):
            p = self.blocks[parent][i]
            self.refs[p] += 1
            self.blocks[child].append(p)
            plan.cell(child, i, p)
        self.lengths[child] = length
        return plan

    def free(self, seq: int) -> Plan:
        """Empties a sequence; pages that no other sequence shares become free."""
        self._seq(seq)
        for p in self.blocks[seq]:
            self._drop(p)
        self.blocks[seq] = []
        self.lengths[seq] = 0
        self._sort_free()
        return Plan()

    def compact(self) -> Plan:
        """Moves the pages with the highest ids into the free pages with the
        lowest, so that the pages in use are 0 .. used - 1."""
        used = self.n_pages - len(self.free_pages)
        holes = sorted(p for p in self.free_pages if p < used)
        movers = [p for p in range(used, self.n_pages) if self.refs[p]]
        plan = Plan(src=movers, dst=holes)
        to = dict(zip(movers, holes))
        for s, mine in enumerate(self.blocks):
            for i, p in enumerate(mine):
                if p in to:
                    mine[i] = to[p]
                    plan.cell(s, i, to[p])
        for a, b in to.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.free_pages = list(range(self.n_pages - 1, used - 1, -1))
        return plan


class PagedKVCache:
    """The FP8 pages of all layers, uint8 [layers, 2, pages, Hk, page, 128] (K
    and V), and the block table int32 [seqs, max_blocks] on ``device``, kept in
    step with a ``PageAllocator``.  The operations work in the order of the
    current stream, like any kernel: use the cache on that stream, or make
    another one wait for it.  Tensors keep their addresses, so captured
    graphs that read them stay valid across operations.  ``k_scales`` /
    ``v_scales``: per layer fp32 [Hk]; ``full_range``: False stores values from
    248 on as the contiguous cache does (ops.paged_kv_write)."""

    def __init__(self, layers: int, n_pages: int, kv_heads: int, page: int, seqs: int, max_blocks: int, device,
                 k_scales: Optional[Sequence[torch.Tensor]] = None, v_scales: Optional[Sequence[torch.Tensor]] = None,
                 full_range: bool = True):
        self.alloc = PageAllocator(n_pages, page, seqs, max_blocks)
        self.layers, self.page = int(layers), int(page)
        self.pool = torch.zeros(layers, 2, n_pages, kv_heads, page, 128, dtype=torch.uint8, device=device)
        self.table = torch.zeros(seqs, max_blocks, dtype=torch.int32, device=device)
        for sc in (k_scales, v_scales):
            if sc is not None and len(sc) != layers:
                raise ValueError(f"{len(sc)} scale tensors for {layers} layers")
        self.k_scales, self.v_scales, self.full_range = k_scales, v_scales, bool(full_range)
        self._views = [(self.pool[i, 0], self.pool[i, 1]) for i in range(layers)]

    @property
    def lengths(self) -> list:
        return self.alloc.lengths

    @property
    def free_count(self) -> int:
        return self.alloc.free_count

    def pages(self, layer: int):
        """(k_pages, v_pages) of a layer, uint8 [pages, Hk, page, 128]."""
        return self._views[layer]

    def codec(self, layer: int) -> dict:
        """Keyword arguments of ops.paged_kv_write for this layer."""
        return dict(self.scales(layer), full_range=self.full_range)

    def scales(self, layer: int) -> dict:
        """Keyword arguments of ops.paged_flash_decode for this layer."""
        return dict(k_scale=None if self.k_scales is None else self.k_scales[layer],
                    v_scale=None if self.v_scales is None else self.v_scales[layer])

    def _run(self, plan: Plan) -> Plan:
        if plan.src:
            ops.kv_copy_pages(self.pool, plan.src, plan.dst)
        if plan.rows:
            ops.kv_table_set(self.table, plan.rows, plan.cols, plan.values)
        return plan

    def extend(self, counts: dict) -> Plan:
        """Room for counts[s] more positions of every sequence s (PageAllocator.extend)."""
        return self._run(self.alloc.extend(counts))

    def fork(self, parent: int, child: int, length: Optional[int] = None) -> Plan:
        return self._run(self.alloc.fork(parent, child, length))

    def free(self, seq: int) -> Plan:
        return self._run(self.alloc.free(seq))

    def compact(self) -> Plan:
        return self._run(self.alloc.compact())
