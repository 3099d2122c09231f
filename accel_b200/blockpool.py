"""tensor.BlockPool (tensor/blockpool.go:46-133) through the C ABI: a host-side free-list page
allocator for a paged KV cache.  It never evicts.

Beyond the reference's pool, pages may be shared between the rows of forked sequences (share / own:
reference counts and copy on write), given back ahead of a sequence's other pages once an attention
window has passed them (trim), and moved together (compact).  The pool only says which pages to copy;
tensor.copy_pages copies them."""
from __future__ import annotations

import ctypes as C
from typing import List, Optional, Sequence, Tuple

import numpy as np

from . import _lib


class BlockPool:
    NONE = 0xffffffff          # a page row's entry whose page has been given back (AB_PAGE_NONE)

    def __init__(self, blocks: int, positions_per_block: int):
        self._h = None
        h = C.c_void_p()
        _lib.check(_lib.lib().ab_blockpool_new(blocks, positions_per_block, C.byref(h)))
        self._h = h
        self._blocks = blocks

    def close(self):
        if getattr(self, "_h", None):
            _lib.lib().ab_blockpool_close(self._h)
            self._h = None

    __del__ = close

    def block_size(self) -> int:
        return _lib.lib().ab_blockpool_block_size(self._h)

    def available(self) -> int:
        return _lib.lib().ab_blockpool_available(self._h)

    def grow(self, pages: Optional[Sequence[int]], n: int) -> List[int]:
        """Pages addressing n positions: the given pages, unmoved, then as many new ones as needed."""
        pages = [] if pages is None else list(pages)
        buf = np.zeros(len(pages) + self._blocks + 1, np.uint32)
        buf[:len(pages)] = pages
        r = _lib.check(_lib.lib().ab_blockpool_grow(self._h, buf.ctypes.data, len(pages), n))
        return [int(x) for x in buf[:r]]

    def free(self, pages: Sequence[int]):
        arr = np.ascontiguousarray(list(pages), dtype=np.uint32)
        _lib.check(_lib.lib().ab_blockpool_free(self._h, arr.ctypes.data, arr.size))

    def positions(self, pages: Sequence[int]) -> int:
        return _lib.lib().ab_blockpool_positions(self._h, len(pages))

    def refs(self, page: int) -> int:
        """How many page rows hold the page; 0 when it is free."""
        return _lib.check(_lib.lib().ab_blockpool_refs(self._h, page))

    def share(self, pages: Sequence[int]) -> List[int]:
        """A second row over the same pages, for a sequence forked off the first: each page has one more
        holder, and goes back to the pool when the last of them frees it."""
        arr = np.ascontiguousarray(list(pages), dtype=np.uint32)
        _lib.check(_lib.lib().ab_blockpool_share(self._h, arr.ctypes.data, arr.size))
        return [int(x) for x in arr]

    def own(self, pages: Sequence[int], start: int, stop: int) -> Tuple[List[int], List[int], List[int]]:
        """Copy on write: the row with its pages that hold the positions [start, stop) held by it alone.
        A page that another row holds too is replaced by a new one; (src, dst) are the copies to make
        (tensor.copy_pages) before the row is read or written."""
        row = list(pages)
        block = self.block_size()
        if not 0 <= start <= stop:
            raise _lib.AccelError(_lib.AB_ERR_INVALID, f"positions [{start}, {stop})")
        a, b = start // block, min((stop + block - 1) // block, len(row))
        if a >= b or start == stop:
            return row, [], []
        part, src, dst = (np.array(row[a:b], np.uint32) for _ in range(3))
        n = _lib.check(_lib.lib().ab_blockpool_own(self._h, part.ctypes.data, part.size, src.ctypes.data, dst.ctypes.data))
        row[a:b] = [int(x) for x in part]
        return row, [int(x) for x in src[:n]], [int(x) for x in dst[:n]]

    def trim(self, pages: Sequence[int], length: int, window: int, sinks: int = 0) -> List[int]:
        """Frees the pages that a sequence of `length` positions will not read again: a query at position
        `length` or later sees the last `window` positions and the first `sinks`.  Their entries become
        BlockPool.NONE, the others stay where they are."""
        if length < 0 or window <= 0 or sinks < 0:
            raise _lib.AccelError(_lib.AB_ERR_INVALID, f"length {length}, window {window}, sinks {sinks}")
        row, block = list(pages), self.block_size()
        lo = max(length + 1 - window, 0)
        a, b = (sinks + block - 1) // block, min(lo // block, len(row))
        if a < b:
            self.free([p for p in row[a:b] if p != self.NONE])
            row[a:b] = [self.NONE] * (b - a)
        return row

    def compact(self, rows: Sequence[Sequence[int]]) -> Tuple[List[List[int]], List[int], List[int]]:
        """Moves the held pages to the lowest numbers.  `rows` are all the page rows in use; returns them
        rewritten, and (src, dst), the copies to make before anything is read through them.  A page that
        is held and in none of the rows is refused: its row could not be rewritten."""
        held = {p for row in rows for p in row if p != self.NONE}
        if len(held) != self._blocks - self.available():
            raise _lib.AccelError(_lib.AB_ERR_INVALID, f"the rows name {len(held)} pages and {self._blocks - self.available()} "
                                  "are held; a compaction moves them all, so it needs every row in use")
        for page in held:
            if self.refs(page) == 0:
                raise _lib.AccelError(_lib.AB_ERR_INVALID, f"a row names block {page}, which is free, and so leaves out one that is held")
        src, dst = np.zeros(self._blocks, np.uint32), np.zeros(self._blocks, np.uint32)
        n = _lib.check(_lib.lib().ab_blockpool_compact(self._h, src.ctypes.data, dst.ctypes.data))
        to = {int(s): int(d) for s, d in zip(src[:n], dst[:n])}
        return [[to.get(p, p) for p in row] for row in rows], list(to), list(to.values())
