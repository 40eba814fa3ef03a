"""Pages of the target's paged K/V cache, kept on the device.

A pool of ``N`` pages serves requests that grow, shrink and leave, and
requests forked from one another (parallel samples, agents on one prompt),
which share the pages of the tokens they have in common:

* ``ref_counts [N]``       — rows that hold each page; 0 is a free page
* ``block_tables [R, C]``  — page of each row's ``block_size`` tokens, -1 none
* ``held [R]``             — pages each row holds (its first entries)

all int32 on the device and owned by the caller; a fresh pool is zeros, -1
and zeros.  The calls are kernels on the current stream and read nothing
back: a bad index is skipped and flagged in the error word, and ``status [2]``
(int32) receives the rows that found no page and the free pages left.  Pages
are handed out lowest id first, rows in call order.  A call names at most 4096
rows; a token's bytes in a cache are a multiple of 16.  The calls change the
pool in place, so two of them on one pool belong on one stream.

The tables are the ``block_table`` of the paged kernels
(:func:`kernels.paged_decode_attention_lse`,
:func:`kernels.shared_prefix_attention_lse`,
:func:`kernels.paged_chunk_attention_scores`).
"""

from __future__ import annotations

import math
from array import array
from collections.abc import Sequence

import torch

from . import _lib

__all__ = ["resize_requests", "fork_requests", "compact_pages", "copy_pages"]


_INT32 = torch.int32


def _pool(ref_counts, block_tables, held):
    """The pool's arguments of every call."""
    if ref_counts.ndim != 1 or block_tables.ndim != 2 or held.ndim != 1:
        raise ValueError("ref_counts must be [pages], block_tables [rows, cols] and held [rows]")
    rows, cols = block_tables.shape
    if held.numel() != rows:
        raise ValueError("held must have one entry per block-table row")
    if not (ref_counts.dtype is _INT32 and block_tables.dtype is _INT32 and held.dtype is _INT32):
        raise ValueError("ref_counts, block_tables and held must be int32")
    stride, step = block_tables.stride()
    if (step != 1 and cols > 1) or not (ref_counts.is_contiguous() and held.is_contiguous()):
        raise ValueError("ref_counts and held must be contiguous, block_tables in contiguous rows")
    if rows == 1:
        stride = cols  # (that of a single row may be anything)
    return (ref_counts.data_ptr(), ref_counts.numel(), block_tables.data_ptr(), rows, stride, cols,
            held.data_ptr())


def _caches(caches: Sequence[torch.Tensor], pages: int):
    """Addresses of the caches (an array to keep), their page size (tokens) and
    a token's bytes."""
    if not len(caches):
        raise ValueError("caches must name at least one tensor")
    first = caches[0]
    if first.ndim < 3:
        raise ValueError("caches must be [pages, block_size, ...]")
    shape, dtype = first.shape, first.dtype
    for t in caches:
        if t.dtype is not dtype or t.shape != shape or not t.is_contiguous():
            raise ValueError("caches must be contiguous tensors of one shape and dtype")
    if shape[0] != pages:
        raise ValueError("caches must have one page per reference count")
    addresses = array("Q", [t.data_ptr() for t in caches])
    # (of the shape: a stride says nothing where a dimension has one entry)
    return addresses, shape[1], math.prod(shape[2:]) * first.element_size()


def _row(t: torch.Tensor, n: int, name: str) -> torch.Tensor:
    if t.ndim != 1 or t.numel() != n:
        raise ValueError(f"{name} must have one entry per request of the call")
    if t.dtype is not _INT32:
        if t.is_floating_point() or t.dtype == torch.bool:
            raise ValueError(f"{name} must be whole numbers")
        if t.dtype is torch.int64:  # (what 32 bits do not hold stays out of range)
            t = t.clamp(-1, 2 ** 31 - 1)
        t = t.to(_INT32)
    return t.contiguous()


def _status(status, like):
    if status is None:
        return like.new_empty(2)
    if status.shape != (2,) or status.dtype is not _INT32 or not status.is_contiguous():
        raise ValueError("status must be int32 [2]")
    return status


def resize_requests(ref_counts: torch.Tensor, block_tables: torch.Tensor, held: torch.Tensor,
                    rows: torch.Tensor, lens: torch.Tensor, *, block_size: int,
                    status: torch.Tensor | None = None) -> torch.Tensor:
    """Give table row ``rows[i]`` the pages of ``lens[i]`` tokens.

    Surplus pages are let go first, those of every row of the call (length 0
    frees a request; a page that another row holds stays), then the missing
    ones are taken from the free pages, rows in call order: the first row
    that does not fit, and every later one that needs pages, keeps what it
    had and is counted in ``status[0]``.  A row outside the table or named
    twice (the first counts), and a length that the table cannot hold, are
    flagged and left alone.

    A row cut back to inside a page that other rows hold after the call keeps
    that page, and it stays theirs: the row's next token would be written over
    their tokens.  Such a row is flagged (``DSB_FLAG_POSITION``); to write on
    from there, fork it at that length instead (:func:`fork_requests` gives the
    child a copy of the started page) and free it.  Returns ``status``."""
    if block_size <= 0:
        raise ValueError("block_size must be positive")
    pool = _pool(ref_counts, block_tables, held)
    n = rows.numel() if rows.ndim == 1 else -1
    rows, lens = _row(rows, n, "rows"), _row(lens, n, "lens")
    device = _lib.device_of(ref_counts, block_tables, held, rows, lens, status)
    status = _status(status, ref_counts)
    _lib.call_on(device, "dsb_resize_requests", *pool, rows.data_ptr(), lens.data_ptr(), n,
                 block_size, status.data_ptr(), _lib.error_flag_ptr(device),
                 _lib.stream_ptr(device))
    return status


def fork_requests(ref_counts: torch.Tensor, block_tables: torch.Tensor, held: torch.Tensor,
                  parents: torch.Tensor, children: torch.Tensor, lens: torch.Tensor,
                  caches: Sequence[torch.Tensor], *,
                  status: torch.Tensor | None = None) -> torch.Tensor:
    """Start table row ``children[i]`` from the first ``lens[i]`` tokens of
    row ``parents[i]``.

    The parent's whole pages are shared (one reference more); the page that
    ``lens[i]`` ends inside is the child's own, the lowest free one, with
    those tokens copied in every cache of ``caches`` (each ``[N, block_size,
    ...]``, all layers' keys and values).  A child must hold no page
    (:func:`resize_requests` to length 0 frees one); one that holds some, is
    named twice (the first counts) or lies outside the table, and a length
    beyond the parent's pages, are flagged and not forked.  Children that
    find no page for their started one are not forked and counted in
    ``status[0]``.  Returns ``status``."""
    pool = _pool(ref_counts, block_tables, held)
    addresses, block_size, token_bytes = _caches(caches, pool[1])
    n = parents.numel() if parents.ndim == 1 else -1
    parents, children = _row(parents, n, "parents"), _row(children, n, "children")
    lens = _row(lens, n, "lens")
    device = _lib.device_of(ref_counts, block_tables, held, parents, children, lens, status, *caches)
    status = _status(status, ref_counts)
    scratch = ref_counts.new_empty(6 * n)  # dsb_fork_scratch_ints
    _lib.call_on(device, "dsb_fork_requests", *pool, parents.data_ptr(), children.data_ptr(),
                 lens.data_ptr(), n, block_size, addresses.buffer_info()[0], len(addresses),
                 token_bytes, status.data_ptr(), scratch.data_ptr(), 6 * n,
                 _lib.error_flag_ptr(device), _lib.stream_ptr(device))
    return status


def compact_pages(ref_counts: torch.Tensor, block_tables: torch.Tensor, held: torch.Tensor,
                  caches: Sequence[torch.Tensor], *,
                  status: torch.Tensor | None = None) -> torch.Tensor:
    """Move the live pages to the front of the pool.

    With ``n`` live pages, the k-th live page with an id of ``n`` or more
    moves to the k-th free page below ``n``, in every cache; the reference
    counts move along and every row's table names the new places.  Pages
    below ``n`` stay where they are.  Returns ``status`` (``status[1]``: the
    free pages, now the last ones)."""
    pool = _pool(ref_counts, block_tables, held)
    addresses, block_size, token_bytes = _caches(caches, pool[1])
    device = _lib.device_of(ref_counts, block_tables, held, status, *caches)
    status = _status(status, ref_counts)
    ints = 1 + 3 * pool[1]  # dsb_compact_scratch_ints
    scratch = ref_counts.new_empty(ints)
    _lib.call_on(device, "dsb_compact_pages", *pool, block_size, addresses.buffer_info()[0],
                 len(addresses), token_bytes, status.data_ptr(), scratch.data_ptr(), ints,
                 _lib.error_flag_ptr(device), _lib.stream_ptr(device))
    return status


def copy_pages(caches: Sequence[torch.Tensor], src: torch.Tensor, dst: torch.Tensor) -> None:
    """``cache[dst[i]] = cache[src[i]]`` for every cache, one launch.

    Pairs with a negative page are skipped, pages outside the caches flagged.
    No page may be both a source and a target of one call, nor a target
    twice: the copies run at the same time."""
    first = caches[0] if len(caches) else None
    if first is None or first.ndim < 3:
        raise ValueError("caches must be [pages, block_size, ...] tensors")
    pages = first.shape[0]
    addresses, block_size, token_bytes = _caches(caches, pages)
    n = src.numel() if src.ndim == 1 else -1
    src, dst = _row(src, n, "src"), _row(dst, n, "dst")
    device = _lib.device_of(src, dst, *caches)
    _lib.call_on(device, "dsb_copy_pages", addresses.buffer_info()[0], len(addresses), pages,
                 block_size * token_bytes, src.data_ptr(), dst.data_ptr(), n,
                 _lib.error_flag_ptr(device), _lib.stream_ptr(device))
