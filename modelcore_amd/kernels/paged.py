"""Block tables and slot maps of a paged KV cache, built on the GPU from request lengths.

A paged cache keeps K and V in a pool of pages of ``page_size`` tokens and, per row, a line of a block
table that names the row's pages. Before a forward ``paged_reserve`` gives every row the pages its new
tokens need and returns where each token goes: its slot (page * page_size + token of the page), which
``rope_norm_scale_append_paged`` writes to, its position, which it rotates by, and the rows' offsets
``cu_seqlens``, which ``flash_attn_paged_with_kvcache`` takes. ``paged_release`` returns the pages of
rows that have ended. Neither reads anything on the host, so both can sit in a captured graph; the
same inputs always give the same pages. ``modelcore_amd.cache.PagedKVCache`` keeps the tables and calls
both.

There is no counterpart in the reference, whose cache reserves T_max positions for every row
(modelcore/cache.py:22-23).
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from modelcore_amd import _ext

__all__ = ["PagedPlan", "paged_reserve", "paged_release", "check_page_size"]


class PagedPlan(NamedTuple):
    """Where a forward's new tokens go (``paged_reserve``)."""
    slots: torch.Tensor       # (total,) int64: page * page_size + token of the page, or -1
    positions: torch.Tensor   # (total,) int32: position within the row, or -1
    cu_seqlens: torch.Tensor  # (rows + 1,) int32: the rows' offsets
    refused: torch.Tensor     # (1,) int32: rows that got no pages, and pages outside the pool


def check_page_size(page_size) -> int:
    page_size = int(page_size)
    if not 16 <= page_size <= 1 << 30 or page_size & (page_size - 1):
        raise ValueError(f"page_size must be a power of two from 16 to 2^30; got {page_size}")
    return page_size


def _check_tables(block_table, cache_seqlens, free_pages, free_count, what):
    _ext.require_rocm(block_table, what=what)
    dev = block_table.device
    _ext.same_device(dev, cache_seqlens=cache_seqlens, free_pages=free_pages, free_count=free_count)
    lines, at = block_table.shape, block_table.stride()
    if block_table.dtype != torch.int32 or len(lines) != 2 or lines[1] < 1 \
            or (at[1] != 1 and lines[1] > 1):
        raise ValueError("block_table must be (rows, max_pages) int32 with contiguous lines; got "
                         f"{tuple(lines)} {block_table.dtype}")
    n, max_pages = lines
    for name, t, shape in (("cache_seqlens", cache_seqlens, (n,)),
                           ("free_pages", free_pages, free_pages.shape[:1]),
                           ("free_count", free_count, (1,))):
        if t.dtype != torch.int32 or t.shape != shape or not t.is_contiguous():
            raise ValueError(f"{name} must be {tuple(shape)} int32, contiguous; got {tuple(t.shape)} "
                             f"{t.dtype}")
    n_pages = free_pages.numel()
    if n_pages < 1:
        raise ValueError("free_pages must have room for every page of the pool")
    # A single line has no stride of its own.
    return n, max_pages, at[0] if n > 1 else max(at[0], max_pages), n_pages, dev


def paged_reserve(block_table, cache_seqlens, new_lens, free_pages, free_count, *, total,
                  page_size) -> PagedPlan:
    """Pages, slots and positions of a forward's new tokens.

    Args:
        block_table: (rows, max_pages) int32, updated in place; -1 where a row holds no page
        cache_seqlens: (rows,) int32, each row's tokens so far (read only)
        new_lens: (rows,) int32, each row's new tokens (0 for a row that has none)
        free_pages: (n_pages,) int32, the stack of free pages, its first free_count numbers
        free_count: (1,) int32, updated in place
        total: the sum of new_lens, known to the host (the forward's token count). Tokens past it
            are not planned; where it is larger, the tokens past the last row's get -1.
        page_size: tokens per page, a power of two from 16 to 2^30

    Returns:
        PagedPlan. A row whose pages the stack does not hold, or that would outgrow its line of the
        table, takes none; its tokens get slot and position -1 and ``refused`` counts it. The length of
        such a row must not move on. A number on the stack that is no page of the pool is counted too, and
        the tokens it was taken for get slot -1.
    """
    n, max_pages, stride, n_pages, dev = _check_tables(block_table, cache_seqlens, free_pages,
                                                       free_count, "paged_reserve")
    _ext.same_device(dev, new_lens=new_lens)
    if new_lens.dtype != torch.int32 or new_lens.shape != (n,):
        raise ValueError(f"new_lens must be ({n},) int32; got {tuple(new_lens.shape)} "
                         f"{new_lens.dtype}")
    new_lens = new_lens.contiguous()
    total, page_size = int(total), check_page_size(page_size)
    if total < 0:
        raise ValueError(f"total must not be negative; got {total}")
    ints = new_lens.new_empty(2 * n + 2 + total)
    cu, refused, positions, scratch = torch.split_with_sizes(ints, [n + 1, 1, total, n])
    slots = new_lens.new_empty(total, dtype=torch.int64)
    with _ext.on_device(dev):
        st = _ext.lib().mcamd_paged_reserve(
            block_table.data_ptr(), stride, cache_seqlens.data_ptr(), new_lens.data_ptr(),
            free_pages.data_ptr(), free_count.data_ptr(), scratch.data_ptr(), cu.data_ptr(),
            slots.data_ptr(), positions.data_ptr(), refused.data_ptr(), n, max_pages,
            n_pages, page_size, total, _ext.stream_handle(dev))
    _ext.check(st, "paged_reserve")
    return PagedPlan(slots, positions, cu, refused)


def _check_release(block_table, cache_seqlens, rows, free_pages, free_count, page_size):
    """Checked mode: every page of the rows that end is one of the pool, held by no other row and not free."""
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("paged_release: checked mode reads the block table on the host and cannot run "
                           "under graph capture; call set_checked(False) first")
    table, lens, width = block_table.tolist(), cache_seqlens.tolist(), block_table.shape[1]
    n_pages = free_pages.numel()
    held = {}
    for b, n in enumerate(lens):
        for page in table[b][:min(-(-max(n, 0) // page_size), width)]:
            held.setdefault(page, []).append(b)
    free = set(free_pages.tolist()[:min(max(free_count.item(), 0), n_pages)])
    for b in rows.tolist():
        if not 0 <= b < len(lens):
            continue
        for page in table[b][:min(-(-max(lens[b], 0) // page_size), width)]:
            if not 0 <= page < n_pages:
                raise IndexError(f"paged_release: page {page} of row {b} is not one of the pool's {n_pages}")
            if page in free or len(held[page]) > 1:
                raise ValueError(f"paged_release: page {page} of row {b} is also "
                                 f"{'free' if page in free else f'held by rows {held[page]}'}")


def paged_release(block_table, cache_seqlens, rows, free_pages, free_count, *, page_size):
    """Rows that have ended give their pages back to the stack, in the order of ``rows`` ((m,)
    int32): their table entries become -1 and their cache_seqlens 0, in place. A row named twice gives
    its pages where it is named first; numbers outside the batch are passed over, and so are table entries
    that are no page of the pool.

    Every page goes onto the stack once for each row that gives it: rows whose lines share pages (which the
    attention only reads) must not be released through more than one of them. Checked mode
    (``flash_attn.set_checked``) reads the tables back and raises where a page is shared, free already or
    outside the pool."""
    n, max_pages, stride, n_pages, dev = _check_tables(block_table, cache_seqlens, free_pages,
                                                       free_count, "paged_release")
    _ext.same_device(dev, rows=rows)
    if rows.dtype != torch.int32 or rows.dim() != 1:
        raise ValueError(f"rows must be (m,) int32; got {tuple(rows.shape)} {rows.dtype}")
    rows, page_size = rows.contiguous(), check_page_size(page_size)
    from modelcore_amd.kernels import flash_attn
    if flash_attn.CHECK_POSITIONS:
        _check_release(block_table, cache_seqlens, rows, free_pages, free_count, page_size)
    with _ext.on_device(dev):
        st = _ext.lib().mcamd_paged_release(
            block_table.data_ptr(), stride, cache_seqlens.data_ptr(), rows.data_ptr(),
            rows.numel(), n, free_pages.data_ptr(), free_count.data_ptr(), max_pages,
            n_pages, page_size, _ext.stream_handle(dev))
    _ext.check(st, "paged_release")
