"""The pages of a 4-bit cache, kept on the device: given to sequences that grow, shared between forks, taken back, and
moved together.

The cache (``attention.cache_pages``) finds a sequence's tokens through its row of a page table.  A ``PagePool`` says
which pages are held:

* ``page_pool(pages, page_size)`` -> a pool whose pages are all free;
* ``reserve(pool, table, lengths, counts)``: pages for each sequence's next tokens, before ``cache_write``;
* ``release(pool, table, first, last)``: pages back, of ended sequences, before a window, or behind dropped tokens;
* ``fork(pool, table, lengths, parents)``: the next batch's rows from the rows of this one: a prompt goes on in many
  ways, beams are kept or dropped, ended sequences leave.  Forks share their parent's finished pages; a page that is not
  full is copied;
* ``compact(pool, table)``: the held pages numbered from 0 on, before a cache is shrunk or handed on;
* ``copy(pages, copies)``: what ``fork`` and ``compact`` ask to be copied, for one cache.  All layers' caches share a
  pool and a table, and each needs this call.

Tables, lengths, counts and parents are int32 tensors on the device.  No call reads them on the host or synchronises, so
all can be captured into a graph (with ``out`` for the results of ``fork``), and none keeps anything between calls.
The free page with the lowest number is given first, so what a pool gives depends on the calls made on it alone.  Where
pages run out, a call goes on without them and says how many it lacked: int32 [1] on the device, to be read whenever the
host looks next.

A pool's calls change it one after another: calls on one pool must be ordered, as on one stream.
"""

from __future__ import annotations

from typing import NamedTuple

import torch
from torch import Tensor

from .attention import TOKENS_PER_TILE, _device, _index, _run
from .runtime import KernelError

MAX_PAGES = 1 << 27
MAX_FORK_SEQUENCES = 8192


class PagePool(NamedTuple):
    """refs [pages]: the table entries that hold each page; free [ceil(pages / 32)]: bit p % 32 of word p / 32 is set
    where refs[p] is 0.  Both int32; page_size in tokens."""

    refs: Tensor
    free: Tensor
    page_size: int


class Fork(NamedTuple):
    """The next rows' table and lengths, the pages to copy [rows, 2] (source and target, then -1), and the pages that
    were lacking [1]."""

    table: Tensor
    lengths: Tensor
    copies: Tensor
    missing: Tensor


def page_pool(pages: int, page_size: int = 64, device: torch.device | str = "cuda") -> PagePool:
    """A pool of `pages` free pages of `page_size` tokens, as cache_pages() makes them."""
    if not 0 < pages <= MAX_PAGES:
        raise KernelError(f"a pool has 1 to {MAX_PAGES} pages, not {pages}")
    if page_size < TOKENS_PER_TILE or page_size & (page_size - 1):
        raise KernelError(f"page_size {page_size} is not a power of two from {TOKENS_PER_TILE} on")
    free = torch.full(((pages + 31) // 32,), -1, dtype=torch.int32)
    if pages % 32:
        free[-1] = (1 << pages % 32) - 1
    return PagePool(torch.zeros(pages, dtype=torch.int32, device=device), free.to(device), page_size)


def _pool(pool: PagePool, what: str) -> tuple[int, int, int, int]:
    """refs, free, pages and page_size, as the library's entries take them."""
    refs, free, page_size = pool
    if refs.dim() != 1 or not 0 < refs.shape[0] <= MAX_PAGES:
        raise KernelError(f"{what} needs a pool as page_pool() makes it")
    count = refs.shape[0]
    _index(refs, count, "refs")
    _index(free, (count + 31) // 32, "free")
    return refs.data_ptr(), free.data_ptr(), count, page_size


def _table(table: Tensor, page_size: int, what: str) -> tuple[int, int]:
    """(sequences, width) of a table."""
    shape = table.shape
    if len(shape) != 2 or table.dtype is not torch.int32 or not table.is_contiguous() or shape[1] == 0:
        raise KernelError(f"{what} needs a contiguous int32 table [sequences, width]")
    if shape[1] * page_size > 1 << 30 or table.numel() >= 1 << 31:
        raise KernelError(f"{what}: a sequence has at most 2**30 tokens, and a table fewer than 2**31 entries")
    return shape[0], shape[1]


def reserve(pool: PagePool, table: Tensor, lengths: Tensor, counts: Tensor) -> Tensor:
    """Gives sequence b the pages for its positions lengths[b] .. lengths[b] + counts[b] - 1, where they are the first to
    use a page and the table has none.  Returns how many got none, for want of free pages or of table entries, at most 2**31 - 1."""
    device = _device(pool.refs, pool.free, table, lengths, counts)
    at = _pool(pool, "reserve")
    sequences, width = _table(table, pool.page_size, "reserve")
    _index(lengths, sequences, "lengths")
    _index(counts, sequences, "counts")
    missing = lengths.new_empty(1)
    _run("ivonar_page_reserve", device, *at, table.data_ptr(), width, lengths.data_ptr(), counts.data_ptr(), sequences,
         missing.data_ptr())
    return missing


def release(pool: PagePool, table: Tensor, first: Tensor | None = None, last: Tensor | None = None) -> None:
    """Sequence b gives back the pages of its slots first[b] .. last[b] - 1 (default: all); their entries become -1.  A
    page that a fork still holds stays held.

    A sequence that has dropped tokens gives back the pages behind its new end, and where that lies within a page that a
    fork holds as well, it has to go through fork() before its next write, which gives it a page of its own."""
    device = _device(pool.refs, pool.free, table, first, last)
    at = _pool(pool, "release")
    sequences, width = _table(table, pool.page_size, "release")
    for tensor, name in ((first, "first"), (last, "last")):
        if tensor is not None:
            _index(tensor, sequences, name)
    _run("ivonar_page_release", device, *at, table.data_ptr(), width, None if first is None else first.data_ptr(),
         None if last is None else last.data_ptr(), sequences)


def fork(pool: PagePool, table: Tensor, lengths: Tensor, parents: Tensor,
         out: tuple[Tensor, Tensor] | None = None) -> Fork:
    """The next batch: row r goes on from row parents[r] of `table` (an empty row where that is none, such as -1).

    The first row of a parent takes over all of its entries; further ones share its finished pages, and get a copy of the
    page that is not full (and none of those reserved behind it).  The first gets one as well where another entry of
    `table` has that page, as after tokens were dropped from a fork.  `table` and `lengths` are used up: rows without a
    child give their pages back.  The copies' pages come from those free before the call; a row that gets none ends with its
    last finished page.  Call copy() with the result's copies for every cache before the next write.
    out: a table [rows, width] and lengths [rows] to write the results into, other tensors than those given."""
    device = _device(pool.refs, pool.free, table, lengths, parents, *(out or ()))
    at = _pool(pool, "fork")
    sequences, width = _table(table, pool.page_size, "fork")
    if sequences > MAX_FORK_SEQUENCES:
        raise KernelError(f"fork takes at most {MAX_FORK_SEQUENCES} sequences, not {sequences}")
    _index(lengths, sequences, "lengths")
    rows = parents.shape[0] if parents.dim() == 1 else -1
    _index(parents, max(rows, 0), "parents")
    if rows * width >= 1 << 31:
        raise KernelError("fork: a table has fewer than 2**31 entries")
    if out is None:
        out = table.new_empty((rows, width)), lengths.new_empty(rows)
    else:
        if _table(out[0], pool.page_size, "fork") != (rows, width):
            raise KernelError(f"out must be a table [{rows}, {width}] and lengths [{rows}]")
        _index(out[1], rows, "the lengths of out")
        if rows and (any(_overlap(to, given) for to in out for given in (table, lengths, parents)) or _overlap(*out)):
            raise KernelError("fork cannot write into the table, lengths or parents that it reads, nor both results alike")
    copies, missing = table.new_empty((rows, 2)), table.new_empty(1)
    _run("ivonar_page_fork", device, *at, table.data_ptr(), width, lengths.data_ptr(), sequences, parents.data_ptr(),
         rows, out[0].data_ptr(), out[1].data_ptr(), copies.data_ptr(), missing.data_ptr())
    return Fork(*out, copies, missing)


def _overlap(a: Tensor, b: Tensor) -> bool:
    return a.data_ptr() < b.data_ptr() + 4 * b.numel() and b.data_ptr() < a.data_ptr() + 4 * a.numel()


def compact(pool: PagePool, table: Tensor) -> tuple[Tensor, Tensor]:
    """(copies [pages / 2, 2], held [1]): the pool's held pages become 0 .. held - 1, in it and in `table`, which has to
    be its only one; those from `held` on take the free numbers below it, both in order.  Call copy() with the copies for
    every cache before its next use."""
    device = _device(pool.refs, pool.free, table)
    at = _pool(pool, "compact")
    sequences, width = _table(table, pool.page_size, "compact")
    copies = table.new_empty((at[2] // 2, 2))
    moved, held = table.new_empty(at[2]), table.new_empty(1)
    _run("ivonar_page_compact", device, *at, table.data_ptr(), width, sequences, copies.data_ptr(), moved.data_ptr(),
         held.data_ptr())
    return copies, held


def copy(pages: Tensor, copies: Tensor) -> None:
    """Copies page copies[i, 0] to page copies[i, 1]; rows with a number outside the pages, such as -1, are skipped.  No
    page may be a source and a target, or a target twice, as in the lists that fork and compact make."""
    device = _device(pages, copies)
    if pages.dim() != 4 or pages.dtype is not torch.uint8 or not pages.is_contiguous() or not pages.numel():
        raise KernelError("copy needs pages as cache_pages() makes them")
    if copies.dim() != 2 or copies.shape[1] != 2 or copies.dtype is not torch.int32 or not copies.is_contiguous():
        raise KernelError("copies must be contiguous int32 [count, 2]")
    if copies.shape[0] >= 1 << 31:
        raise KernelError("copy takes fewer than 2**31 copies")
    if copies.data_ptr() & 7:
        copies = copies.clone()
    page_bytes = pages.numel() // pages.shape[0]
    if page_bytes % 16 or pages.data_ptr() & 15:
        raise KernelError("copy needs pages as cache_pages() makes them, that start on 16 bytes")
    _run("ivonar_page_copy", device, pages.data_ptr(), pages.shape[0], page_bytes, copies.data_ptr(), copies.shape[0])
