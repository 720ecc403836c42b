"""Keys and values in pages: which page holds what (PageTable, host only), and the pools on the device
with the tables that the kernels read (PagedCache).

A sequence holds a slot of the batch and a list of pages; position t is in its page t // page_size.
Forked sequences share the pages that are full (a page is freed when its last holder leaves); the
partly filled last page is copied at the fork, so a page that rows are still appended to has one
holder.  The reference has no counterpart (one contiguous cache per layer, ops.py:533-576).
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

import numpy as np

from . import _lib
from . import kernels as K
from .device import DeviceBuffer, DeviceSlice, PinnedBuffer


class OutOfPages(RuntimeError):
    """The pool has no page left for what was asked; nothing was changed."""


class PageTable:
    """Page ids, lengths and holders of up to `batch` sequences over `num_pages` pages.  Operations
    that move contents return lists (src, dst) of pages to copy before anything else is done."""

    def __init__(self, num_pages: int, page_size: int, batch: int, max_pages: int):
        if min(num_pages, page_size, batch, max_pages) < 1:
            raise ValueError("a page table needs at least one page, position, sequence and page per sequence")
        self.num_pages, self.page_size, self.batch, self.max_pages = int(num_pages), int(page_size), int(batch), int(max_pages)
        self.table = np.full((self.batch, self.max_pages), -1, np.int32)
        self.lengths = np.zeros(self.batch, np.int32)
        self.holders = np.zeros(self.num_pages, np.int32)
        self.live = np.zeros(self.batch, bool)
        self._free = list(range(self.num_pages - 1, -1, -1))       # the lowest page is taken first

    def free_pages(self) -> int:
        return len(self._free)

    def _check(self, slot: int) -> int:
        slot = int(slot)
        if not 0 <= slot < self.batch or not self.live[slot]:
            raise ValueError(f"no sequence in slot {slot}")
        return slot

    def _pages(self, slot: int) -> int:
        return -(-int(self.lengths[slot]) // self.page_size)

    def _take(self) -> int:
        page = self._free.pop()
        self.holders[page] = 1
        return page

    def _drop(self, page: int) -> None:
        self.holders[page] -= 1
        if self.holders[page] == 0:
            self._free.append(int(page))

    def open(self) -> int:
        """A slot for a new, empty sequence."""
        for slot in range(self.batch):
            if not self.live[slot]:
                self.live[slot] = True
                self.lengths[slot] = 0
                return slot
        raise OutOfPages("every slot of the batch is taken")

    def extend(self, slot: int, tokens: int = 1) -> None:
        """Makes the sequence `tokens` longer; kv_append fills the new positions."""
        slot, tokens = self._check(slot), int(tokens)
        if tokens < 0:
            raise ValueError("a sequence is not extended by less than nothing")
        have, need = self._pages(slot), -(-(int(self.lengths[slot]) + tokens) // self.page_size)
        if need > self.max_pages:
            raise OutOfPages(f"a sequence has at most {self.max_pages} pages")
        if need - have > len(self._free):
            raise OutOfPages(f"{need - have} pages wanted, {len(self._free)} free")
        for i in range(have, need):
            self.table[slot, i] = self._take()
        self.lengths[slot] += tokens

    def fork(self, slot: int) -> tuple[int, list, list]:
        """A second sequence with the same tokens: (its slot, src, dst)."""
        slot = self._check(slot)
        n, part = self._pages(slot), int(self.lengths[slot]) % self.page_size
        if part and not self._free:
            raise OutOfPages("no page for the copy of the last one")
        other = self.open()
        src, dst = [], []
        for i in range(n):
            page = int(self.table[slot, i])
            if i == n - 1 and part:
                src.append(page)
                page = self._take()
                dst.append(page)
            elif page >= 0:
                self.holders[page] += 1
            self.table[other, i] = page
        self.lengths[other] = self.lengths[slot]
        return other, src, dst

    def close(self, slot: int) -> None:
        """Ends a sequence; pages that no other holds are free again."""
        slot = self._check(slot)
        for page in self.table[slot, : self._pages(slot)]:
            if page >= 0:
                self._drop(int(page))
        self.table[slot] = -1
        self.lengths[slot] = 0
        self.live[slot] = False

    def trim(self, slot: int, window: int, sinks: int = 0) -> int:
        """Frees the pages that attention with this window and these sinks cannot see any more, now or
        for a longer sequence; returns how many the sequence gave up."""
        slot = self._check(slot)
        if window < 1 or sinks < 0:
            raise ValueError("trim needs a window")
        start, count = int(self.lengths[slot]) - int(window), 0
        for i in range(-(-int(sinks) // self.page_size), max(0, start) // self.page_size):
            page = int(self.table[slot, i])
            if page >= 0:
                self._drop(page)
                self.table[slot, i] = -1
                count += 1
        return count

    def compact(self) -> tuple[list, list]:
        """Moves the pages in use to the lowest ids: (src, dst).  Afterwards pages from used_pages()
        on hold nothing."""
        used = np.flatnonzero(self.holders)
        n = len(used)
        holes = np.flatnonzero(self.holders[:n] == 0)
        src = used[used >= n]
        dst = holes[: len(src)]
        to = np.arange(self.num_pages, dtype=np.int32)
        to[src] = dst
        held = self.table >= 0
        self.table[held] = to[self.table[held]]
        self.holders[dst] = self.holders[src]
        self.holders[src] = 0
        self._free = list(range(self.num_pages - 1, n - 1, -1))
        return src.tolist(), dst.tolist()

    def used_pages(self) -> int:
        return int(np.count_nonzero(self.holders))


class PagedCache:
    """The pages of all layers on the device, [layer][page][kv head][slot][element] for keys and for
    values (8-bit pages: and their scales), with the page table and lengths that the kernels read."""

    def __init__(self, layers: int, kv_heads: int, dh: int, num_pages: int, page_size: int = 16, batch: int = 1,
                 max_pages: Optional[int] = None, dtype: str = "bf16", device: Optional[int] = None):
        if dtype not in K.DTYPES:
            raise ValueError(f"unknown element type {dtype!r}")
        self.layers, self.kv_heads, self.dh, self.dtype = int(layers), int(kv_heads), int(dh), dtype
        self.pages = PageTable(num_pages, page_size, batch, num_pages if max_pages is None else max_pages)
        self.itemsize = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1}[dtype]
        self.page_elems = self.kv_heads * int(page_size) * self.dh
        size = self.layers * int(num_pages) * self.page_elems * self.itemsize
        self.k, self.v = DeviceBuffer(size, device, zero=True), DeviceBuffer(size, device, zero=True)
        self.scales = None
        if dtype == "i8":
            rows = self.layers * int(num_pages) * self.kv_heads * int(page_size) * 4
            self.scales = (DeviceBuffer(rows, device, zero=True), DeviceBuffer(rows, device, zero=True))
        self._bytes = (self.pages.table.nbytes, self.pages.lengths.nbytes)
        self.table, self.lengths = DeviceBuffer(self._bytes[0], device, zero=True), DeviceBuffer(self._bytes[1], device, zero=True)
        # two staging areas take turns: one may still be on its way while the other is written
        self._staging = [PinnedBuffer(sum(self._bytes)) for _ in range(2)]
        self._events = []
        for _ in self._staging:
            e = C.c_void_p()
            _lib.call("mira_cuda_event_create", C.byref(e))
            self._events.append([e, False])
        self._turn = 0
        self._sent = np.full_like(self.pages.table, -2)
        self._regions = K.page_regions(self._region_list())

    def _region_list(self) -> list:
        n, ps = self.pages.num_pages, self.pages.page_size
        pages = self.page_elems * self.itemsize
        out = [K.PageRegion(b, page_bytes=pages, page_stride=pages, planes=self.layers, plane_stride=n * pages) for b in (self.k, self.v)]
        if self.scales:
            rows = self.kv_heads * ps * 4
            out += [K.PageRegion(b, page_bytes=rows, page_stride=rows, planes=self.layers, plane_stride=n * rows) for b in self.scales]
        return out

    def layer(self, i: int) -> K.PagedKV:
        """Layer i's pages, as kv_append and paged_attention take them."""
        if not 0 <= i < self.layers:
            raise ValueError(f"no layer {i}")
        ps, n = self.pages.page_size, self.pages.num_pages
        at = i * n * self.page_elems * self.itemsize
        st = (self.page_elems, ps * self.dh, self.dh, 1)
        more = {}
        if self.scales:
            views = [K.View(DeviceSlice(b, i * n * self.kv_heads * ps * 4), (self.kv_heads * ps, ps, 1, 1)) for b in self.scales]
            more = dict(k_scale=views[0], v_scale=views[1])
        return K.PagedKV(num_pages=n, page_size=ps, kv_heads=self.kv_heads, dh=self.dh, dtype=self.dtype,
                         k=K.View(DeviceSlice(self.k, at), st), v=K.View(DeviceSlice(self.v, at), st), batch=self.pages.batch,
                         table=self.table, table_ld=self.pages.max_pages, max_pages=self.pages.max_pages,
                         lengths=self.lengths, **more)

    def open(self) -> int:
        return self.pages.open()

    def extend(self, slot: int, tokens: int = 1) -> None:
        self.pages.extend(slot, tokens)

    def close(self, slot: int) -> None:
        self.pages.close(slot)

    def trim(self, slot: int, window: int, sinks: int = 0) -> int:
        return self.pages.trim(slot, window, sinks)

    def fork(self, slot: int) -> int:
        """A second sequence with the same tokens."""
        other, src, dst = self.pages.fork(slot)
        if src:
            K.page_copy(self._regions, self.pages.num_pages, src, dst)
        return other

    def compact(self) -> int:
        """Moves the pages in use to the front of the pools; returns how many moved."""
        src, dst = self.pages.compact()
        if src:
            K.page_copy(self._regions, self.pages.num_pages, src, dst)
        return len(src)

    def sync_tables(self) -> None:
        """Sends lengths, and the page table if it changed, to the device, in order with the launches
        (call after open / extend / fork / close / trim / compact, before the next launch)."""
        table = not np.array_equal(self._sent, self.pages.table)
        stage, (event, used) = self._staging[self._turn], self._events[self._turn]
        if used:
            _lib.call("mira_cuda_event_sync", event)
        nt, nl = self._bytes
        host = stage.view((nt + nl,), np.uint8)
        host[nt:] = self.pages.lengths.view(np.uint8)
        _lib.call("mira_cuda_h2d", C.c_void_p(self.lengths.ptr), C.c_void_p(stage.ptr + nt), C.c_size_t(nl))
        if table:
            host[:nt] = self.pages.table.reshape(-1).view(np.uint8)
            _lib.call("mira_cuda_h2d", C.c_void_p(self.table.ptr), C.c_void_p(stage.ptr), C.c_size_t(nt))
            self._sent[...] = self.pages.table
        _lib.call("mira_cuda_event_record", event)
        self._events[self._turn][1] = True
        self._turn ^= 1

    def free(self) -> None:
        """Gives the device and staging memory back."""
        _lib.call("mira_cuda_sync")
        for e, _ in self._events:
            _lib.call("mira_cuda_event_destroy", e)
        self._events = []
        for b in [self.k, self.v, self.table, self.lengths, *(self.scales or ()), *self._staging]:
            b.close()
