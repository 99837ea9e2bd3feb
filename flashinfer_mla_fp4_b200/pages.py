"""The care of a paged cache: copying, allocating, forking, freeing and compacting pages, on the device.

The reference leaves the pages to its caller.  A serving program that samples several continuations of a prompt, keeps a prefix for later
requests or runs for days needs the rest of what a paged cache is for:

* ``copy_pages``      pages copied to other numbers, in every layer;
* ``FP4MLAPagePool``  reference counts over the pages of one or more layers: ``allocate`` pages for growing requests, ``fork`` a request into
  others that share its full pages, ``free`` requests, ``compact`` the pages in use to the low end of the pool.

Everything is decided on the device, from counts, lengths and tables in device memory: no call synchronises, and all can be recorded in a CUDA
graph.  What a call could not do is reported by ``check_status()``.  A page moves with its scales and, in caches that have
them, its summary.
"""
from __future__ import annotations

import ctypes as C
import os
from typing import Optional, Sequence

import torch

from . import _cabi
from .adapter import FP4MLAPagedCache
from .api_log import api_logged
from .sparse import check_cache, check_summary, check_tables, check_tensor


def _layers(caches: Sequence[FP4MLAPagedCache]):
    """(array of the C ABI, pages, page size, device, the tensors) of caches that hold a page of the same number each."""
    caches = list(caches)
    if not caches:
        raise ValueError("at least one cache is needed")
    pages, page_size = check_cache(caches[0].kv_cache, caches[0].kv_cache_sf)
    dev = caches[0].kv_cache.device
    array, kept = (_cabi.PageLayer * len(caches))(), []
    for i, c in enumerate(caches):
        if check_cache(c.kv_cache, c.kv_cache_sf) != (pages, page_size) or c.kv_cache.device != dev:
            raise ValueError("the caches of a pool must share the number of pages, the page size and the device")
        array[i].kv_cache, array[i].kv_cache_sf = c.kv_cache.data_ptr(), c.kv_cache_sf.data_ptr()
        kept += [c.kv_cache, c.kv_cache_sf]
        if c.summary is not None:
            check_summary(c.summary, c.summary_sf, pages, dev)
            array[i].summary, array[i].summary_sf = c.summary.data_ptr(), c.summary_sf.data_ptr()
            kept += [c.summary, c.summary_sf]
    starts = [t.data_ptr() for t in kept]
    if len(set(starts)) != len(starts):
        raise ValueError("a cache is given twice")
    return array, pages, page_size, dev, kept


@api_logged
def copy_pages(caches: Sequence[FP4MLAPagedCache], src: torch.Tensor, dst: torch.Tensor) -> None:
    """Copy page ``src[i]`` to page ``dst[i]`` in every cache (rows, scales, summary), for all i at once.

    ``src`` and ``dst``: int32 [n] on the caches' device; pairs with a page outside the pool (-1, say) are skipped.  No page may be named twice in
    ``dst``, nor in both lists: the copies run side by side and would race (``MLA_FP4_VALIDATE=1`` checks it, and synchronises)."""
    array, pages, page_size, dev, _ = _layers(caches)
    check_tensor("src", src, torch.int32, (None,), dev)
    check_tensor("dst", dst, torch.int32, (src.shape[0],), dev)
    if os.environ.get("MLA_FP4_VALIDATE", "0") not in ("", "0"):
        pairs = [(s, d) for s, d in zip(src.tolist(), dst.tolist()) if 0 <= s < pages and 0 <= d < pages and s != d]
        to = [d for _, d in pairs]
        if len(set(to)) != len(to) or set(to) & {s for s, _ in pairs}:
            raise ValueError("copy_pages: a page is named twice among dst, or both in src and in dst")
    if src.numel() == 0:
        return
    with torch.cuda.device(dev):
        _cabi.check(_cabi.lib.mla_fp4_copy_pages(array, len(array), pages, page_size, src.data_ptr(), dst.data_ptr(), src.numel(),
                                                 torch.cuda.current_stream(dev).cuda_stream))


class FP4MLAPagePool:
    """Pages of one or more layers with reference counts: ``refcounts`` int32 [pages], 0 = free.

    ``caches``: the layers' caches, one page number meaning the same page in each; they are kept, and their tensors must stay the ones they
    were.  The block tables (int32 [rows, max_pages]) and lengths (int32 [rows], the tokens that a row holds) are the program's own device
    tensors; lists of rows are int32 device tensors, negative entries padding.  New pages are the free ones of the lowest numbers, in the
    order in which they are asked for.  Calls on a pool belong on one stream, or ordered by events: they change the counts.
    """

    def __init__(self, caches: Sequence[FP4MLAPagedCache]) -> None:
        self.caches = list(caches)
        self._array, self.num_pages, self.page_size, self.device, self._kept = _layers(self.caches)
        self._address = C.addressof(self._array)
        self.refcounts = torch.zeros(self.num_pages, dtype=torch.int32, device=self.device)
        self._status = torch.zeros(8, dtype=torch.int32, device=self.device)

    def _native(self, what: int, block_tables, seq_lens, x, y=None):
        """The common form of a call, checked and launched natively; None: nothing was done."""
        return _cabi.native.pool(what, self._address, len(self._array), self.page_size, self.num_pages, self.refcounts, self._status,
                                  block_tables, seq_lens, x, y)

    def num_free(self) -> int:
        """Free pages (synchronises)."""
        return int((self.refcounts <= 0).sum())

    def _args(self, block_tables: torch.Tensor, seq_lens: torch.Tensor, count: int):
        check_tables(block_tables, seq_lens, self.device)
        rows, width = block_tables.shape
        if rows > 1 and block_tables.stride(0) < width:
            raise ValueError("the rows of block_tables must not overlap")
        check_tensor("refcounts", self.refcounts, torch.int32, (self.num_pages,), self.device)
        need = _cabi.pool_workspace_bytes(self.num_pages, rows, count)
        workspace = torch.empty(need, dtype=torch.int8, device=self.device)
        a = _cabi.PoolArgs()
        a.layers, a.num_layers, a.page_size, a.num_pages = self._array, len(self._array), self.page_size, self.num_pages
        a.refcounts, a.block_tables, a.block_table_stride = self.refcounts.data_ptr(), block_tables.data_ptr(), block_tables.stride(0)
        a.width, a.rows, a.seq_lens = width, rows, seq_lens.data_ptr()
        a.workspace, a.workspace_bytes, a.status = workspace.data_ptr(), need, self._status.data_ptr()
        a.stream = torch.cuda.current_stream(self.device).cuda_stream
        return a, workspace

    @api_logged
    def allocate(self, block_tables: torch.Tensor, seq_lens: torch.Tensor, new_lens: torch.Tensor) -> None:
        """Give each row the pages that ``new_lens`` (int32 [rows]) tokens take beyond those for ``seq_lens``; the lengths stay as they are.

        Rows are served in order.  One that no longer fits into the pool, or into its block-table row, gets nothing, and what there is stays for
        the rows behind it.  Take the new lengths over into ``seq_lens`` before the next call on the pool: until then no row has the new pages, so
        ``free`` or a second ``allocate`` would lose them, ``fork`` would not share them and ``compact`` would leave their table entries on the old numbers.  A length may
        be lowered within the row's last page if no fork shares that (a full one may be shared); a page behind the new end would be the row's no longer, and nobody's."""
        if self._native(0, block_tables, seq_lens, new_lens) is not None:
            return
        check_tables(block_tables, seq_lens, self.device)
        check_tensor("new_lens", new_lens, torch.int32, (block_tables.shape[0],), self.device)
        if block_tables.shape[0] == 0:
            return
        with torch.cuda.device(self.device):
            a, _workspace = self._args(block_tables, seq_lens, 0)
            _cabi.check(_cabi.lib.mla_fp4_pool_allocate(C.byref(a), new_lens.data_ptr()))

    @api_logged
    def fork(self, block_tables: torch.Tensor, seq_lens: torch.Tensor, parents: torch.Tensor, children: torch.Tensor) -> None:
        """Make row ``children[i]`` what row ``parents[i]`` is: full pages are shared, a last page that is not full is copied in every layer.

        A child's row must be empty (length 0); a parent may have many children.  A fork for which the pool has no page, into a row that is not
        empty, or of a child that the list has named before, is not made."""
        if self._native(1, block_tables, seq_lens, parents, children) is not None:
            return
        check_tensor("parents", parents, torch.int32, (None,), self.device)
        check_tensor("children", children, torch.int32, (parents.shape[0],), self.device)
        if parents.numel() == 0:
            return
        with torch.cuda.device(self.device):
            a, _workspace = self._args(block_tables, seq_lens, parents.numel())
            _cabi.check(_cabi.lib.mla_fp4_pool_fork(C.byref(a), parents.data_ptr(), children.data_ptr(), parents.numel()))

    @api_logged
    def free(self, block_tables: torch.Tensor, seq_lens: torch.Tensor, rows: torch.Tensor) -> None:
        """Take a reference from every page of the rows and set their lengths to 0 (a row that is named twice is freed once)."""
        if self._native(2, block_tables, seq_lens, rows) is not None:
            return
        check_tensor("rows", rows, torch.int32, (None,), self.device)
        if rows.numel() == 0:
            return
        with torch.cuda.device(self.device):
            a, _workspace = self._args(block_tables, seq_lens, rows.numel())
            _cabi.check(_cabi.lib.mla_fp4_pool_free(C.byref(a), rows.data_ptr(), rows.numel()))

    @api_logged
    def compact(self, block_tables: torch.Tensor, seq_lens: torch.Tensor, remap: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Move the n pages in use to the numbers below n: the i-th of those numbered n or more into the i-th free one below n, in every layer.

        Reference counts and the block tables' entries (as far as ``seq_lens`` says) follow.  Returns ``remap`` int32 [pages]: the new number of
        each page, -1 for one that was free, for whatever else names pages."""
        done = self._native(3, block_tables, seq_lens, remap)
        if done is not None:
            return done
        if remap is None:
            remap = torch.empty(self.num_pages, dtype=torch.int32, device=self.device)
        else:
            check_tensor("remap", remap, torch.int32, (self.num_pages,), self.device)
        with torch.cuda.device(self.device):
            a, _workspace = self._args(block_tables, seq_lens, 0)
            _cabi.check(_cabi.lib.mla_fp4_pool_compact(C.byref(a), remap.data_ptr()))
        return remap

    def check_status(self) -> None:
        """Raise for what the calls since the last check could not do (synchronises)."""
        code, which = (int(x) for x in self._status[:2].cpu())
        if code:
            self._status.zero_()
            if code == _cabi.POOL_OUT_OF_PAGES:
                raise RuntimeError(f"mla_fp4 page pool: no page left for entry {which}")
            raise ValueError(f"mla_fp4 page pool: entry {which} names a row that is out of range, too short, not empty, named twice or already free")


__all__ = ["FP4MLAPagePool", "copy_pages"]
