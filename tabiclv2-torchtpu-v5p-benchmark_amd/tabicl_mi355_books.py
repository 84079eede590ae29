"""The books of a paged K/V cache on the GPU: which page holds which rows, kept by kernels instead of the host, so that a step
of a service (pages for new rows, the rows into them, attention) can be captured in a graph and replayed while its requests
grow. PagedIclKVCache keeps them on the host; these functions are for callers with a pool of their own.

  * paged_reserve (op tabicl::paged_reserve): pages for the rows that each request gets, from a stack of free pages;
  * paged_slots (op tabicl::paged_slots): where each row of a packed batch goes, and where each request's rows start in it;
  * paged_append_packed (ops tabicl::paged_append_slots, paged_append_q8): such rows into their places;
  * paged_release (op tabicl::paged_release): pages behind the rows that stay, back to the stack.

free [pages] int32 is the stack, free_count [1] int32 how many pages lie on it (the top one last); pages = free.numel() is the
pool's number of pages: an entry of the table outside [0, pages) holds no page. No page may stand in the table or on the stack
twice. No counterpart in the reference."""
from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor

import tabicl_mi355_native as _nat
import tabicl_mi355_paged8 as _p8
import tabicl_mi355_pool as _pool


def _free_args(free: Tensor, free_count: Tensor, dev: int) -> None:
    if free.dtype is not torch.int32 or free.dim() != 1 or not free.is_contiguous() or free.get_device() != dev:
        raise ValueError("free must be a contiguous int32 [pages] tensor on the table's device")
    if free_count.dtype is not torch.int32 or free_count.numel() != 1 or free_count.get_device() != dev:
        raise ValueError("free_count must be an int32 tensor of one entry on the table's device")


def _own_rows(table: Tensor) -> None:
    if table.shape[0] > 1 and table.stride(0) < table.shape[1]:
        raise ValueError("the rows of a table that is written to must not overlap")


def _reserve_launch(table: Tensor, lengths: Tensor, count: Tensor, free: Tensor, free_count: Tensor, page_rows: int,
                    granted: Tensor) -> None:
    t, N = _pool.table_args(table, lengths)
    dev = table.get_device()
    _pool.counts(count, N, "count")
    _free_args(free, free_count, dev)
    _own_rows(table)
    if lengths.get_device() != dev or count.get_device() != dev:
        raise ValueError("table, lengths and count must be on one device")
    if _pool.elsewhere(dev, table):
        with torch.cuda.device(dev):
            return _reserve_launch(table, lengths, count, free, free_count, page_rows, granted)
    ws, ptr, nbytes = _pool.workspace(int(_nat.load().tabicl_paged_books_workspace_bytes(N)), "tabicl_paged_reserve", table)
    _nat.call("tabicl_paged_reserve", *t, lengths.data_ptr(), count.data_ptr(), free.data_ptr(), free_count.data_ptr(),
              granted.data_ptr(), free.numel(), page_rows, N, ptr, nbytes, _nat.stream_of(table))


@torch.library.custom_op("tabicl::paged_reserve", mutates_args=("table", "free_count"))
def _paged_reserve(table: Tensor, lengths: Tensor, count: Tensor, free: Tensor, free_count: Tensor, page_rows: int) -> Tensor:
    """See paged_reserve."""
    granted = torch.empty(table.shape[0], dtype=torch.int32, device=table.device)
    _reserve_launch(table, lengths, count, free, free_count, page_rows, granted)
    return granted


@_paged_reserve.register_fake
def _(table, lengths, count, free, free_count, page_rows):  # noqa: ANN001
    return table.new_empty(table.shape[0])


def paged_reserve(table: Tensor, lengths: Tensor, count: Tensor, free: Tensor, free_count: Tensor, page_rows: int) -> Tensor:
    """Gives each request n pages for count[n] rows behind its lengths[n] (int32 [N] on the GPU): the entries of table
    [N, max_pages] from the first page behind row lengths[n] to that of the last new row that hold no page get pages from the top
    of the stack, request by request, as far as they go. Returns granted [N] int32: how many of the rows have a place (all,
    or those before the first page that was not to be had; none, where row lengths[n] joins a page that the table does not have).
    lengths and count stay as they are. In place: table, free_count."""
    if _nat.direct(table, lengths, count, free, free_count):
        granted = None
        if _nat.DIRECT is not None:
            granted = _nat.DIRECT.reserve(table, lengths, count, free, free_count, int(page_rows), _nat.stream_of(table))
        if granted is None:
            granted = torch.empty(table.shape[:1], dtype=torch.int32, device=table.device)
            _reserve_launch(table, lengths, count, free, free_count, int(page_rows), granted)
        torch.autograd.graph.increment_version((table, free_count))
        return granted
    return torch.ops.tabicl.paged_reserve(table, lengths, count, free, free_count, int(page_rows))


def _release_launch(table: Tensor, lengths: Tensor, free: Tensor, free_count: Tensor, page_rows: int) -> None:
    t, N = _pool.table_args(table, lengths)
    dev = table.get_device()
    _free_args(free, free_count, dev)
    _own_rows(table)
    if lengths.get_device() != dev:
        raise ValueError("table and lengths must be on one device")
    if _pool.elsewhere(dev, table):
        with torch.cuda.device(dev):
            return _release_launch(table, lengths, free, free_count, page_rows)
    ws, ptr, nbytes = _pool.workspace(int(_nat.load().tabicl_paged_books_workspace_bytes(N)), "tabicl_paged_release", table)
    _nat.call("tabicl_paged_release", *t, lengths.data_ptr(), free.data_ptr(), free_count.data_ptr(), free.numel(), page_rows, N,
              ptr, nbytes, _nat.stream_of(table))


@torch.library.custom_op("tabicl::paged_release", mutates_args=("table", "free", "free_count"))
def _paged_release(table: Tensor, lengths: Tensor, free: Tensor, free_count: Tensor, page_rows: int) -> None:
    """See paged_release."""
    _release_launch(table, lengths, free, free_count, page_rows)


@_paged_release.register_fake
def _(table, lengths, free, free_count, page_rows):  # noqa: ANN001
    return None


def paged_release(table: Tensor, lengths: Tensor, free: Tensor, free_count: Tensor, page_rows: int) -> None:
    """Puts the pages behind row lengths[n] of each request back on the stack, -1 in their place: rows that were withdrawn or
    evicted, or (lengths 0) a request that is done. The last request's last page goes first, so that a release of what a
    reserve gave out leaves the stack as it was. In place: table, free, free_count."""
    if _nat.direct(table, lengths, free, free_count):
        if _nat.DIRECT is None or not _nat.DIRECT.release(table, lengths, free, free_count, int(page_rows), _nat.stream_of(table)):
            _release_launch(table, lengths, free, free_count, int(page_rows))
        torch.autograd.graph.increment_version((table, free, free_count))
    else:
        torch.ops.tabicl.paged_release(table, lengths, free, free_count, int(page_rows))


def _slots(table: Tensor, lengths: Tensor, count: Tensor, total: int, pages: int, page_rows: int) -> tuple[Tensor, Tensor]:
    t, N = _pool.table_args(table, lengths)
    dev = table.get_device()
    _pool.counts(count, N, "count")
    if lengths.get_device() != dev or count.get_device() != dev:
        raise ValueError("table, lengths and count must be on one device")
    if _pool.elsewhere(dev, table):
        with torch.cuda.device(dev):
            return _slots(table, lengths, count, total, pages, page_rows)
    slots = torch.empty(total, dtype=torch.int64, device=table.device)
    starts = torch.empty(N + 1, dtype=torch.int32, device=table.device)
    _nat.call("tabicl_paged_slots", *t, lengths.data_ptr(), count.data_ptr(), slots.data_ptr(), starts.data_ptr(), total, pages,
              page_rows, N, _nat.stream_of(table))
    return slots, starts


@torch.library.custom_op("tabicl::paged_slots", mutates_args=())
def _paged_slots(table: Tensor, lengths: Tensor, count: Tensor, total: int, pages: int, page_rows: int) -> tuple[Tensor, Tensor]:
    """See paged_slots."""
    return _slots(table, lengths, count, total, pages, page_rows)


@_paged_slots.register_fake
def _(table, lengths, count, total, pages, page_rows):  # noqa: ANN001
    return table.new_empty(total, dtype=torch.int64), table.new_empty(table.shape[0] + 1)


def paged_slots(table: Tensor, lengths: Tensor, count: Tensor, total: int, pages: int, page_rows: int) -> tuple[Tensor, Tensor]:
    """Where the rows of a packed batch go (count[0] rows of request 0, then those of request 1, ...): slots [total] int64, page
    * page_rows + the row in it, for the row that becomes row lengths[n] + t of its request, or -1 where it has no page;
    starts [N + 1] int32, the running sums of the counts (they must add up to less than 2^31). total may be more than the rows
    there are (a captured graph's size): the places behind them are -1."""
    if total < 0:
        raise ValueError(f"total must not be negative, got {total}")
    if _nat.direct(table, lengths, count):
        if _nat.DIRECT is not None:
            r = _nat.DIRECT.slots(table, lengths, count, int(total), int(pages), int(page_rows), _nat.stream_of(table))
            if r is not None:
                return r
        return _slots(table, lengths, count, int(total), int(pages), int(page_rows))
    return torch.ops.tabicl.paged_slots(table, lengths, count, int(total), int(pages), int(page_rows))


def _append_launch(k_pages: Tensor, v_pages: Tensor, slots: Tensor, k: Tensor, v: Tensor) -> None:
    shape, st, dev = k_pages.shape, k_pages.stride(), k_pages.get_device()
    if len(shape) != 4 or v_pages.shape != shape or v_pages.stride() != st or k_pages.dtype is not v_pages.dtype:
        raise ValueError(f"k_pages and v_pages must be [pages, H, page_rows, D] of one layout and dtype, got {tuple(shape)} and "
                         f"{tuple(v_pages.shape)}")
    P, H, R, D = shape
    if st[3] != 1 or st[2] != D or (st[1] != R * D and H > 1):
        raise ValueError("a page [H, page_rows, D] must be contiguous")
    if k.dim() != 3 or v.shape != k.shape or k.shape[1:] != (H, D):
        raise ValueError(f"k and v must be [total, {H}, {D}], got {tuple(k.shape)} and {tuple(v.shape)}")
    if k.dtype is not k_pages.dtype or v.dtype is not k_pages.dtype:
        raise ValueError(f"paged_append_packed expects {k_pages.dtype} (cast before appending)")
    if slots.dtype is not torch.int64 or slots.shape != k.shape[:1] or not slots.is_contiguous():
        raise ValueError(f"slots must be a contiguous int64 tensor of {k.shape[0]} entries")
    if any(t.get_device() != dev for t in (v_pages, slots, k, v)):
        raise ValueError("slots, k, v and the pool must be on one device")
    code = _nat.dtype_code(k.dtype)
    if _pool.elsewhere(dev, k_pages):
        with torch.cuda.device(dev):
            return _append_launch(k_pages, v_pages, slots, k, v)
    es = k.element_size()
    k, _, kh, kr = _pool.rows16(k.unsqueeze(0).transpose(1, 2), es)
    v, _, vh, vr = _pool.rows16(v.unsqueeze(0).transpose(1, 2), es)
    _nat.call("tabicl_paged_append_slots", k_pages.data_ptr(), v_pages.data_ptr(), P, st[0] if P > 1 else H * R * D, R,
              slots.data_ptr(), k.data_ptr(), v.data_ptr(), k.shape[2], H, D, kr, kh, vr, vh, code, _nat.stream_of(k))


@torch.library.custom_op("tabicl::paged_append_slots", mutates_args=("k_pages", "v_pages"))
def _paged_append_slots(k_pages: Tensor, v_pages: Tensor, slots: Tensor, k: Tensor, v: Tensor) -> None:
    """See paged_append_packed."""
    _append_launch(k_pages, v_pages, slots, k, v)


@_paged_append_slots.register_fake
def _(k_pages, v_pages, slots, k, v):  # noqa: ANN001
    return None


def paged_append_packed(k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, count: Tensor, k: Tensor, v: Tensor,
                        slots: Tensor, starts: Tensor, scales: Optional[Tensor] = None) -> None:
    """Packed rows k, v [total, H, D] (any strides with a contiguous last dim) to the places that paged_slots found for
    them with the same table, lengths and count; rows without one are left out. lengths is read, not changed. With scales: a
    pool of 8-bit codes, whose pages take their rows as paged_append's do."""
    if scales is not None or k_pages.dtype in _pool.CODES:
        _p8.append(k_pages, v_pages, table, lengths, k, v, count, starts, scales)
    elif _nat.direct(k_pages, v_pages, slots, k, v):
        if _nat.DIRECT is None or not _nat.DIRECT.append_slots(k_pages, v_pages, slots, k, v, _nat.stream_of(k)):
            _append_launch(k_pages, v_pages, slots, k, v)
        torch.autograd.graph.increment_version((k_pages, v_pages))
    else:
        _pool.no_grad("paged_append_packed", k_pages, v_pages, k, v)
        torch.ops.tabicl.paged_append_slots(k_pages, v_pages, slots, k, v)
