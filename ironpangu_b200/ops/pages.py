"""Pages of key-value caches that sequences share, on the device (``csrc/kernels/pages.cu``): a pool whose pages are taken, shared by forks, packed and given back by kernels,
so that a step which forks its sequences needs no host and runs inside a CUDA graph, and copies of pages between caches.

Where a pool's call finds a slot or a length out of range, a slot named twice that it would give pages, or fewer free pages than it needs, it changes nothing and sets a bit of
``status`` (:meth:`PagePool.check` raises for it); :func:`copy` skips what is out of range and copies the rest. Nothing waits for the host. Calls of one pool, and kernels that read or write its pages, are ordered by the caller: one stream, or
events. ``runtime/paged_state.py`` is the other way to hold pages, with leases on the host."""
from __future__ import annotations

import ctypes as C
from typing import List, Optional

import torch

from . import _lib
from ._lib import call_on

I32 = torch.int32
BAD_INDEX, NO_PAGES = 4, 8          # IFAB_STATUS_* of common.cuh
MAX_SLOTS = 8192


class IfabPageSet(C.Structure):
    """Mirror of ``struct IfabPageSet`` in ``csrc/kernels/ifab_kernels.h``."""

    _fields_ = [("ptrs", C.c_void_p), ("row_bytes", C.c_void_p), ("caches", C.c_int32), ("pages", C.c_int32), ("page_tokens", C.c_int32), ("max_row_bytes", C.c_int64)]


class IfabPagePool(C.Structure):
    """Mirror of ``struct IfabPagePool``."""

    _fields_ = [("set", IfabPageSet), ("table", C.c_void_p), ("lengths", C.c_void_p), ("refs", C.c_void_p), ("free_bits", C.c_void_p), ("work", C.c_void_p),
                ("status", C.c_void_p), ("slots", C.c_int32), ("max_pages", C.c_int32)]


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(f"pages: {what}")


class PageSet:
    """Caches whose page ``i`` belongs together: contiguous tensors ``[pages, page_tokens, ...]`` of any types on one device, a row a multiple of 16 bytes."""

    def __init__(self, caches: List[torch.Tensor]):
        _need(len(caches) > 0, "no caches")
        self.caches = list(caches)                    # kept: the kernels go by their addresses
        t = caches[0]
        _need(all(c.is_cuda and c.device == t.device and c.dim() >= 2 and c.shape[:2] == t.shape[:2] and c.is_contiguous() for c in caches),
              "caches must be contiguous [pages, page_tokens, ...] on one device, with as many pages and rows each")
        self.pages, self.page_tokens, self.device, self.index = t.shape[0], t.shape[1], t.device, t.get_device()
        _need(self.pages > 0 and self.page_tokens > 0, "caches without pages")
        _need(self.pages < 1 << 30 and self.page_tokens < 1 << 20, "caches too large")
        self.row_bytes = [c[0, 0].numel() * c.element_size() for c in caches]
        _need(all(r > 0 and r % 16 == 0 for r in self.row_bytes) and all(c.data_ptr() % 16 == 0 for c in caches), "a row must be a multiple of 16 bytes, on 16 bytes")
        self._ptrs = torch.tensor([c.data_ptr() for c in caches], dtype=torch.int64, device=t.device)
        self._rows = torch.tensor(self.row_bytes, dtype=torch.int64, device=t.device)
        self.status = torch.zeros(1, dtype=I32, device=t.device)
        self.status_ptr = self.status.data_ptr()
        self.desc = IfabPageSet(self._ptrs.data_ptr(), self._rows.data_ptr(), len(caches), self.pages, self.page_tokens, max(self.row_bytes))
        self.ref = C.byref(self.desc)

    def check(self) -> None:
        """Raises when a copy into this set met an index that is out of range (waits for the device)."""
        if int(self.status):
            self.status.zero_()
            raise IndexError("pages: an index out of range was skipped")

    def _list(self, t: torch.Tensor, what: str, n: int) -> int:
        if not (t.dtype is I32 and t.shape == (n,) and t.get_device() == self.index and (n < 2 or t.stride(0) == 1)):
            _need(t.dim() == 1 and t.dtype == I32 and t.device == self.device and (t.numel() < 2 or t.stride(0) == 1), f"{what} must be a contiguous int32 list on {self.device}")
            _need(False, f"{what}: {t.numel()} entries beside {n}")
        return t.data_ptr()


def copy(src: PageSet, dst: PageSet, src_ids: torch.Tensor, dst_ids: torch.Tensor, rows: Optional[torch.Tensor] = None) -> None:
    """Page ``dst_ids[i]`` of every cache of ``dst`` becomes page ``src_ids[i]`` of ``src``, its first ``rows[i]`` rows only where ``rows`` is given. The sets have rows of
    the same sizes and may be one set; pages that are written must differ from one another and from those that are read. Entries out of range are skipped and reported in
    ``dst.status``."""
    if src is not dst and not (src.row_bytes == dst.row_bytes and src.page_tokens == dst.page_tokens and src.device == dst.device):
        _need(False, "the sets' pages are not alike")
    n = src_ids.numel()
    a, b = src._list(src_ids, "src_ids", n), src._list(dst_ids, "dst_ids", n)
    call_on(src.index, "ifab_pages_copy", src.ref, dst.ref, a, b, None if rows is None else src._list(rows, "rows", n), n, dst.status_ptr)


class PagePool:
    """The pages of ``caches`` for ``slots`` sequences of up to ``max_pages`` pages each. ``table`` ``[slots, max_pages]`` (-1: none) is what attention kernels take as
    their page table; ``lengths`` ``[slots]``: positions a slot holds pages for; ``refs`` ``[pages]``: entries of the table that name a page. Free pages are taken lowest first, in
    the order of a call's list."""

    def __init__(self, caches: List[torch.Tensor], *, slots: int, max_pages: int):
        self.pages = s = PageSet(caches)
        # positions, and the table's entries, are counted in 32 bits
        _need(1 <= slots <= MAX_SLOTS and max_pages >= 1 and (max_pages + 1) * s.page_tokens < 1 << 31 and slots * max_pages < 1 << 31,
              f"{slots} slots of {max_pages} pages are not supported")
        self.slots, self.max_pages, self.page_tokens, self.device = slots, max_pages, s.page_tokens, s.device
        self.index = s.index
        i32 = lambda *shape, v=0: torch.full(shape, v, dtype=I32, device=s.device)
        self.table, self.lengths, self.refs, self.live = i32(slots, max_pages, v=-1), i32(slots), i32(s.pages), i32(1)
        words = (s.pages + 31) // 32
        self._bits = i32(words, v=-1)
        if s.pages % 32:
            self._bits[-1] = (1 << s.pages % 32) - 1
        self._work = i32(_lib.load().ifab_pages_work_words(slots, max_pages, s.pages))
        self.status = i32(1)
        self.desc = IfabPagePool(s.desc, self.table.data_ptr(), self.lengths.data_ptr(), self.refs.data_ptr(), self._bits.data_ptr(), self._work.data_ptr(),
                                 self.status.data_ptr(), slots, max_pages)
        self.ref = C.byref(self.desc)

    def check(self) -> None:
        """Raises when a call was refused on the device since the last check (waits for the device): IndexError where a list named a slot out of range, a slot twice or a length
        that no slot can hold, OverflowError where pages lacked (where both happened, the next check raises for the other)."""
        bits = int(self.status)
        if bits & BAD_INDEX:
            self.status.bitwise_and_(~BAD_INDEX)
            raise IndexError("pages: a list of slots named one out of range or twice, or a length that no slot can hold")
        if bits:
            self.status.zero_()
            raise OverflowError("pages: the pool had fewer free pages than a call needed")

    def extend(self, slots: torch.Tensor, tokens: torch.Tensor) -> None:
        """Slot ``slots[i]`` gets pages for positions below ``tokens[i]`` (where it has them already nothing changes). A slot may be named once. All or nothing."""
        n = slots.numel()
        a, b = self.pages._list(slots, "slots", n), self.pages._list(tokens, "tokens", n)
        if n > self.slots:
            _need(False, f"{n} entries for {self.slots} slots")
        call_on(self.index, "ifab_pages_extend", self.ref, a, b, n)

    def fork(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        """Slot ``dst[i]`` becomes what slot ``src[i]`` was before the call; what it held before is given back. ``dst`` names a slot once, ``src`` as often as wanted, and a slot
        may be in both. Whole pages are shared. A partly filled page, which its sequence goes on writing, stays with the first child of a slot that is itself replaced; every
        other child gets a page of its own with the rows in use copied. All or nothing."""
        n = src.numel()
        a, b = self.pages._list(src, "src", n), self.pages._list(dst, "dst", n)
        if n > self.slots:
            _need(False, f"{n} entries for {self.slots} slots")
        call_on(self.index, "ifab_pages_fork", self.ref, a, b, n)

    def free(self, slots: torch.Tensor, below: Optional[torch.Tensor] = None) -> None:
        """All pages of the slots are given back, or with ``below`` the whole pages all of whose positions lie below ``below[i]`` (a window has passed them); those
        entries of the table are -1 then. A page goes back to the pool when no other slot holds it. A slot may be named more than once (the furthest ``below`` counts). All or
        nothing: a list with a slot out of range or a negative ``below`` frees no page."""
        n = slots.numel()
        a, b = self.pages._list(slots, "slots", n), None if below is None else self.pages._list(below, "below", n)
        call_on(self.index, "ifab_pages_free", self.ref, a, b, n)

    def compact(self) -> None:
        """Live pages move into the lowest places - the first one that lies too high into the first hole, and so on - in all caches, and the table follows; their
        number lands in ``live``."""
        call_on(self.index, "ifab_pages_compact", self.ref, self.live.data_ptr())
