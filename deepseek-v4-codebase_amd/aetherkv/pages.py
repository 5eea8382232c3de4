"""The pages of paged per-head caches (aetherkv.paged): given to sequences, shared by forks, copied before they are written,
released, and moved together.

A PagePool serves the caches of all layers, which share one page table: it counts for every page the table entries that hold
it, and keeps what append_tokens and evict_by_weight need, which write to the pages of the slots they fill:

  reserve   the slots that are about to be written lie in pages of their sequence's own
  fork      rows take over other rows' pages without copying them (answers to one prompt, beams, cached prefixes)
  release   the pages behind a sequence's kept slots are free again
  compact   the pages in use are the pool's first ones, so that what lies behind them can be given up

Tables (of at most 4096 rows) and counts are device tensors and nothing synchronises, so these calls can be captured in a graph.
A table entry of -1 (any outside the pool) holds no page.  The calls change the table and the pool's counts: those of one pool
run one after another (on one stream, or with events between).  Rows of a table need not be sequences of the batch: a prefix that
is kept for later is a row, and attention takes the rows before it, page_table[:B].
"""
from __future__ import annotations

from array import array
from typing import Optional, Sequence

import torch

from . import _lib
from .paged import PagedKVCache, _counts, _given, _one_device

_SEGMENT = 4096  # bytes of a page's tensor that a wave copies at a time


class PagePool:
    """The pages of `caches` (one per layer, with the same pages and page size), none in use; refs: existing counts int32 [pages],
    used in place."""

    def __init__(self, caches: Sequence[PagedKVCache], *, refs: Optional[torch.Tensor] = None):
        caches = tuple(caches)
        if not caches:
            raise ValueError("PagePool needs a cache")
        head = caches[0]
        if head.pages < 1:
            raise ValueError("PagePool needs caches with pages")
        for c in caches[1:]:
            if c.pages != head.pages or c.page_size != head.page_size or c._index != head._index:
                raise RuntimeError(f"the caches of a pool need the same pages, page size and device, got {c.pages} x {c.page_size} on {c.device} beside "
                                   f"{head.pages} x {head.page_size} on {head.device}")
        self.caches, self.pages, self.page_size, self.device, self._index = caches, head.pages, head.page_size, head.device, head._index
        # (zeros in one allocation: counts where none are given, the kernels' marks, what reserve lacked)
        n, own = self.pages, refs is None
        zeros = torch.zeros((3 if own else 2) * n + 1, dtype=torch.int32, device=self.device)
        if own:
            refs = zeros[2 * n + 1:]
        elif refs.dtype != torch.int32 or refs.shape != (n,) or not refs.is_contiguous() or refs.get_device() != self._index:
            raise RuntimeError(f"refs must be contiguous int32 [{n}] on {self.device}, got {refs.dtype} {tuple(refs.shape)} on {refs.device}")
        self._refs, self._marks, self._lacking = refs, zeros[:2 * n].view(2, n), zeros[2 * n:2 * n + 1]
        rows = array("q")  # where a page's bytes lie: address of page 0, step, bytes
        for c in caches:
            for t in c._tensors:
                page, at = t.stride(0) * t.element_size(), t.data_ptr()
                for off in range(0, page, _SEGMENT):
                    rows.extend((at + off, page, min(_SEGMENT, page - off)))
        self._segments = (torch.frombuffer(rows, dtype=torch.int64) if rows else torch.empty(0, dtype=torch.int64)).to(self.device)
        self._args = (self._segments.data_ptr(), len(rows) // 3)

    refs = property(lambda self: self._refs)

    @property
    def lacking(self) -> torch.Tensor:
        """int32 [1]: pages that reserve could not give since it was last set to 0.  Their entries are -1: what is written to their
        slots is lost, and so are the tokens that a row had in a page it shared (the page's other holders keep them).  A later reserve
        gives such an entry an empty page, not those tokens: the sequence has to end, or be filled again."""
        return self._lacking

    def unused(self) -> torch.Tensor:
        """The number of pages that no table entry holds (a tensor: nothing waits).  Not within a captured graph: a torch reduction
        may clear its scratch there by a memset node, which does not hold over replays."""
        if _lib._capturing():
            raise RuntimeError("unused() is no call for a captured graph: take it between replays")
        return (self._refs <= 0).sum()

    def _table(self, page_table: torch.Tensor):
        """The table is written: int32, contiguous (a conversion would be written instead)."""
        if page_table.dim() != 2 or page_table.dtype is not torch.int32 or not page_table.is_contiguous():
            raise RuntimeError(f"page_table must be contiguous int32 [B, max_pages], got {page_table.dtype} {tuple(page_table.shape)} {page_table.stride()}")
        return page_table.shape

    def workspace(self, rows: int, max_pages: int, forks: int = 0) -> torch.Tensor:
        """Workspace of the calls on a table [rows, max_pages]."""
        n = _lib.pool_ws_bytes(int(rows), int(max_pages), int(forks), self.pages)
        return torch.empty(n, dtype=torch.uint8, device=self.device)

    def reserve(self, page_table: torch.Tensor, filled: torch.Tensor, wanted: torch.Tensor, *, first: Optional[torch.Tensor] = None,
                workspace: Optional[torch.Tensor] = None) -> None:
        """Slots first[b] .. wanted[b] - 1 of every sequence are about to be written; its slots before filled[b] hold tokens.

        Each entry of those slots' pages that holds none gets an unused page; one that holds a page which other entries hold too
        gets an unused page with a copy of it (if it has filled slots), unless the call gives pages to all those entries, of which
        the last (by row) keeps it.  Unused pages are taken from the lowest on, in the order of the entries.  first (default:
        filled): zeros before evict_by_weight, which writes anywhere.  filled, wanted, first int32 [B].

        Where the pool is out of pages an entry becomes -1, `lacking` counts it, and what the entry shared is lost to its row.  That
        does not happen where unused(), read with the tokens of the step before, is at least the number of entries that the call
        covers (one per row for a step's token).  A row waits by wanted[b] <= first[b]: it takes no page and keeps what it shares, as
        long as nothing is appended to it or evicted."""
        B, W = self._table(page_table)
        _one_device(self._index, page_table, filled, wanted, first, workspace)
        filled, wanted = _counts("filled", filled, B), _counts("wanted", wanted, B)
        first = None if first is None else _counts("first", first, B)
        need = _lib.pool_ws_bytes(B, W, 0, 0) if workspace is None else 0
        dev = self.device
        with _lib.on_device(dev):
            stream = _lib.raw_stream(dev)
            ws = _given(workspace) if workspace is not None else _lib.workspace(need, dev, stream)
            rc = _lib.hot("aekv_pool_reserve")(
                page_table.data_ptr(), B, W, filled.data_ptr(), wanted.data_ptr(), None if first is None else first.data_ptr(), self.page_size,
                self._refs.data_ptr(), self._marks.data_ptr(), self._lacking.data_ptr(), self.pages, *self._args,
                None if ws is None else ws.data_ptr(), 0 if ws is None else ws.numel(), stream)
        if rc:
            _lib.check(rc, "aekv_pool_reserve")

    def release(self, page_table: torch.Tensor, keep: torch.Tensor) -> None:
        """Every sequence lets go of its pages behind the first keep[b] slots (int32 [B]; 0: of all)."""
        B, W = self._table(page_table)
        _one_device(self._index, page_table, keep)
        keep = _counts("keep", keep, B)
        dev = self.device
        with _lib.on_device(dev):
            rc = _lib.hot("aekv_pool_release")(page_table.data_ptr(), B, W, keep.data_ptr(), self.page_size, self._refs.data_ptr(), self.pages,
                                               _lib.raw_stream(dev))
        if rc:
            _lib.check(rc, "aekv_pool_release")

    def fork(self, page_table: torch.Tensor, filled: torch.Tensor, source: torch.Tensor, target: torch.Tensor, *,
             workspace: Optional[torch.Tensor] = None) -> None:
        """Row target[j] lets go of its pages and holds those of the first filled[source[j]] slots of row source[j] as well (source
        and target int32 [n], filled int32 [B]).

        All rows are read as they were before the call, so that beams can change places; a row to itself stays as it is; of
        several forks to one row the last counts; one from or to a row outside the table is skipped.  `filled` is only read: the
        caller sets filled[target] = filled[source] (and a tracker's rows likewise), and reserves before it writes."""
        B, W = self._table(page_table)
        _one_device(self._index, page_table, filled, source, target, workspace)
        if source.dim() != 1:
            raise RuntimeError(f"source must be int32 [n], got {source.dtype} {tuple(source.shape)}")
        n = source.size(0)
        filled, source, target = _counts("filled", filled, B), _counts("source", source, n), _counts("target", target, n)
        need = _lib.pool_ws_bytes(0, W, n, 0) if workspace is None else 0
        dev = self.device
        with _lib.on_device(dev):
            stream = _lib.raw_stream(dev)
            ws = _given(workspace) if workspace is not None else _lib.workspace(need, dev, stream)
            rc = _lib.hot("aekv_pool_fork")(
                page_table.data_ptr(), B, W, filled.data_ptr(), source.data_ptr(), target.data_ptr(), n, self.page_size, self._refs.data_ptr(),
                self.pages, None if ws is None else ws.data_ptr(), 0 if ws is None else ws.numel(), stream)
        if rc:
            _lib.check(rc, "aekv_pool_fork")

    def compact(self, *page_tables: torch.Tensor, workspace: Optional[torch.Tensor] = None) -> None:
        """Moves the pages in use to the pool's first ones: with n in use, the k-th unused page below n takes the k-th one in use
        from n on, in every layer.  page_tables: all tables that hold the pool's pages."""
        if not page_tables:
            raise RuntimeError("compact needs every table that holds the pool's pages")
        for t in page_tables:
            self._table(t)
        _one_device(self._index, *page_tables, workspace)
        first, *others = page_tables
        dev = self.device
        with _lib.on_device(dev):
            stream = _lib.raw_stream(dev)
            # (several calls use the workspace where there are other tables: a kept one could serve another call between them)
            ws = _given(workspace) if workspace is not None else self.workspace(0, 0) if others else _lib.workspace(_lib.pool_ws_bytes(0, 0, 0, self.pages), dev, stream)
            at, size = ws.data_ptr(), ws.numel()
            rc = _lib.hot("aekv_pool_compact")(first.data_ptr(), first.numel(), self._refs.data_ptr(), self.pages, *self._args, at, size, stream)
            if rc:
                _lib.check(rc, "aekv_pool_compact")
            for t in others:
                _lib.check(_lib.lib().aekv_pool_renumber(t.data_ptr(), t.numel(), self.pages, at, size, stream), "aekv_pool_renumber")
