"""The pages of the paged cache (larder_amd.attention) as a pool on the GPU that tables share. Every call queues its kernels on
the current stream and none waits for the GPU, so that a step's pages are given, shared and freed between its other launches
(and captured in a graph with them).

    take_pages(refs, table, lens, cu)     the places that the newest rows fall into get pages of their own
    copy_pages(cache, src, dst)           codes and scales of pages, as take_pages and compact_pages ask for
    fork_pages(refs, table, parents)      a table whose sequences go on from those of another
    free_pages(refs, table, keep)         sequences cut to their first tokens, or ended
    compact_pages(refs, *tables)          held pages moved into the lowest numbers

A pool is refs int32 [pages], zeros at first: how many places of the tables hold a page. A table int32 [sequences, places] lists
each sequence's pages in order and has -1 wherever it holds none, behind its last page too. One pool and its tables serve the
caches of all layers: what a layer's cache has to copy comes as a list of pairs. Everything has one result, whatever the
order in which threads run: the lowest free pages go to the first sequences' first places.

A page that several sequences hold is only read; before rows are appended, take_pages gives a sequence a page of its own in the
place of one that it shares, and the pair to copy. A step is then

    src, dst, lacking = take_pages(refs, table, lens, cu)         # lens with the rows about to be appended
    for cache in caches: copy_pages(cache, src, dst)
    append_rows(cache, ..., table, lens, cu), attend_rows / chunk_rows(..., table, lens, cu)

The host does not see what these tensors hold: numbers outside the pool count as no page, wrong counts give pages of no meaning,
and no other memory is touched.
"""
import functools

import torch

from . import _lib, attention
from .attention import _MOST, _device, _ints, _launch, _refuse

__all__ = ["compact_pages", "copy_pages", "fork_pages", "free_pages", "take_pages"]


def _pool(fn, refs, table):
    """(pages, sequences, places): the pool's and a table's sizes, both written in place."""
    if refs.dtype is not torch.int32 or refs.dim() != 1 or refs.shape[0] == 0 or not refs.is_contiguous():
        _refuse(fn, f"refs is int32 [pages], contiguous, not {refs.dtype} {list(refs.shape)}")
    if table.dtype is not torch.int32 or table.dim() != 2 or table.shape[1] == 0 or not table.is_contiguous():
        _refuse(fn, f"table is int32 [sequences, places], contiguous, not {table.dtype} {list(table.shape)}")
    pages, (n, places) = refs.shape[0], table.shape
    if pages > _MOST or n > _MOST or places > _MOST:
        _refuse(fn, f"{pages} pages, {n} sequences of {places} places are more than an int counts")
    return pages, n, places


def _page(fn, page):
    if page not in (32, 64, 128):
        _refuse(fn, f"pages of {page} tokens (32, 64 and 128 are served)")


@functools.lru_cache(maxsize=1024)
def _take_workspace(*sizes):
    return _lib.lib().lmoe_pages_take_workspace_bytes(*sizes)


@functools.lru_cache(maxsize=64)
def _compact_workspace(pages):
    return _lib.lib().lmoe_pages_compact_workspace_bytes(pages)


def take_pages(refs, table, lens, cu=None, page=64):
    """Gives every place of the table that the newest rows fall into a page that is its sequence's alone: the lowest free one
    (refs 0 when the call begins) where it has none, or where its page has other holders. lens, cu as append_rows takes them (the
    rows counted in lens; one row a sequence where cu is None), page: the cache's tokens a page. refs and table are written in place.

    (src, dst, lacking), int32 [sequences] each: the pages to copy before the rows are appended, where a sequence had shared
    a page that holds tokens before them (-1: none; a sequence has one at most), and how many of its places found no page left.
    Those hold -1 and what they shared is no longer theirs: append_rows writes nothing there, and such a sequence is cut
    (free_pages) and taken up again when there is room. But a page that all of its holders would leave so stays with the last of
    those that found none, and is its own. Tokens past the table's places have none, and lack none."""
    fn = "take_pages"
    pages, n, places = _pool(fn, refs, table)
    _page(fn, page)
    lens = _ints(fn, "lens", lens, n)
    if cu is not None:
        cu = _ints(fn, "cu", cu, n + 1)
    dev = _device(fn, refs, table, lens, cu)
    src, dst, lacking = refs.new_empty((3, n)).unbind(0)
    if n:
        need = _take_workspace(n, places, pages)
        ws = refs.new_empty(need, dtype=torch.uint8)
        _launch(dev, "lmoe_pages_take", refs.data_ptr(), pages, table.data_ptr(), n, places, lens.data_ptr(),
                None if cu is None else cu.data_ptr(), page, src.data_ptr(), dst.data_ptr(), lacking.data_ptr(), ws.data_ptr(),
                need)
    return src, dst, lacking


def copy_pages(cache, src, dst):
    """Copies the pages src[i] of a cache to dst[i] (int32 [pairs]; a pair with a number outside the cache is left out): codes and
    scales, of keys and values. No page is in dst twice, or in both."""
    fn = "copy_pages"
    pages, heads, page, width, *codes = attention._cache(fn, cache)
    if src.dim() != 1:
        _refuse(fn, f"src is int32 [pairs], not {src.dtype} {list(src.shape)}")
    n = src.shape[0]
    if n > _MOST:
        _refuse(fn, f"{n} pairs are more than an int counts")
    src, dst = _ints(fn, "src", src, n), _ints(fn, "dst", dst, n)
    dev = _device(fn, *cache, src, dst)
    if n:
        _launch(dev, "lmoe_pages_copy", *codes, pages, page, heads, width, src.data_ptr(), dst.data_ptr(), n)


def fork_pages(refs, table, parents):
    """A new table int32 [len(parents), places] whose sequence i goes on from sequence parents[i] (int32) of the old one and shares
    its pages; parents outside the table begin empty. The old table's places are given back in the same call: sequences
    that no parent names end, sequences named once have only moved, and the old table is not used again. Beams are reordered,
    samples drawn from one prompt and finished sequences dropped by one call; lens follows as lens[parents.long()], with 0 for
    those that begin empty."""
    fn = "fork_pages"
    pages, n, places = _pool(fn, refs, table)
    if parents.dim() != 1:
        _refuse(fn, f"parents is int32 [sequences], not {parents.dtype} {list(parents.shape)}")
    if parents.shape[0] > _MOST:
        _refuse(fn, f"{parents.shape[0]} new sequences are more than an int counts")
    parents = _ints(fn, "parents", parents, parents.shape[0])
    dev = _device(fn, refs, table, parents)
    out = table.new_empty((parents.shape[0], places))
    if n or out.shape[0]:
        _launch(dev, "lmoe_pages_fork", refs.data_ptr(), pages, table.data_ptr(), n, places, parents.data_ptr(), out.shape[0],
                out.data_ptr())
    return out


def free_pages(refs, table, keep, page=64):
    """Cuts each sequence to its first keep[b] (int32 [sequences]) tokens: places behind them are given back and hold -1; 0 ends
    the sequence, and as many tokens as it has cut nothing but pages that no token has reached. In place."""
    fn = "free_pages"
    pages, n, places = _pool(fn, refs, table)
    _page(fn, page)
    keep = _ints(fn, "keep", keep, n)
    dev = _device(fn, refs, table, keep)
    if n:
        _launch(dev, "lmoe_pages_free", refs.data_ptr(), pages, table.data_ptr(), n, places, keep.data_ptr(), page)


def compact_pages(refs, *tables):
    """Renumbers the held pages into the lowest numbers, so that what lies behind them can be given up: those past the first
    `used` (as many as are held) take the free numbers among these, both in order. refs and every table of the pool are
    written in place. (src, dst, used): the pairs that copy_pages has to copy in every cache, int32 [pages / 2] with -1 behind
    the last one, and used int32 [1]."""
    fn = "compact_pages"
    if not tables:
        _refuse(fn, "no table")
    sizes = [_pool(fn, refs, t) for t in tables]
    dev = _device(fn, refs, *tables)
    pages = refs.shape[0]
    src, dst = (refs.new_empty(max(pages // 2, 1)) for _ in range(2))
    used, to = refs.new_empty(1), refs.new_empty(pages)
    need = _compact_workspace(pages)
    ws = refs.new_empty(need, dtype=torch.uint8)
    _launch(dev, "lmoe_pages_compact", refs.data_ptr(), pages, src.data_ptr(), dst.data_ptr(), used.data_ptr(), to.data_ptr(),
            ws.data_ptr(), need)
    for t, (_, n, places) in zip(tables, sizes):
        if n:
            _launch(dev, "lmoe_pages_renumber", t.data_ptr(), n, places, pages, used.data_ptr(), to.data_ptr())
    return src, dst, used
