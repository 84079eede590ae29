"""Attention over selected pages of a paged K/V cache on MI355X: a test row reads the pages of its table whose keys can give
it the largest scores, and leaves the others alone.

  * paged_bounds (op tabicl::paged_bounds): the largest and the smallest value of each dim of a page's keys, in int8 with one
    power of two per page and head: bounds [pages, H, 2, D] int8 (0: largest, rounded up; 1: smallest, rounded down),
    bound_scales [pages, H] fp32;
  * paged_select (op tabicl::paged_select): the pages of largest bound for each query row and K/V head;
  * paged_sparse_attention (ops tabicl::paged_sparse_attn, paged_sparse_attn_out): attention over the pages that an index lists.

The bound of a page for a query row: the sum over the dims of u_d hi_d where u_d > 0 and u_d lo_d where it is not (the larger
of the two), times the page's scale; u is the query row in int8 (one power of two for the heads of a group), the largest over
the group's heads counts. Whole numbers below 2^24 times a power of two: the
selection is the same on every run and machine. Pools in bf16, fp32, and e4m3 or int8 with their scales
(tabicl_mi355_paged8). No counterpart in the reference, whose queries read the whole cache."""
from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor

import tabicl_mi355_native as _nat
import tabicl_mi355_pool as _pool


def _check_bounds(bounds: Tensor, bound_scales: Tensor, P: int, H: int, D: int, dev: int) -> None:
    if bounds.dtype is not torch.int8 or bounds.shape != (P, H, 2, D) or not bounds.is_contiguous() or bounds.data_ptr() & 15 \
            or bounds.get_device() != dev:
        raise ValueError(f"bounds must be a contiguous int8 [{P}, {H}, 2, {D}] tensor that starts on 16 bytes, on the table's device, "
                         f"got {bounds.dtype} {tuple(bounds.shape)}")
    if bound_scales.dtype is not torch.float32 or bound_scales.shape != (P, H) or not bound_scales.is_contiguous() \
            or bound_scales.get_device() != dev:
        raise ValueError(f"bound_scales must be a contiguous float32 [{P}, {H}] tensor on the table's device, got "
                         f"{bound_scales.dtype} {tuple(bound_scales.shape)}")


def _bounds_launch(k_pages: Tensor, table: Tensor, lengths: Tensor, bounds: Tensor, bound_scales: Tensor,
                   start: Optional[Tensor], rows: int, scales: Optional[Tensor]) -> None:
    pool, H, D, N, dev = _pool.pool_args(k_pages, k_pages, table, lengths)
    fmt = _pool.pool_format(k_pages, scales, dev)
    _check_bounds(bounds, bound_scales, pool[0], H, D, dev)
    if start is not None:
        _pool.counts(start, N, "start")
        if start.get_device() != dev:
            raise ValueError("start must be on the table's device")
    if _pool.elsewhere(dev, k_pages):
        with torch.cuda.device(dev):
            return _bounds_launch(k_pages, table, lengths, bounds, bound_scales, start, rows, scales)
    _nat.call("tabicl_paged_bounds", k_pages.data_ptr(), None if scales is None else scales.data_ptr(), *pool, lengths.data_ptr(),
              None if start is None else start.data_ptr(), min(rows, pool[5] * pool[2]), bounds.data_ptr(),
              bound_scales.data_ptr(), N, H, D, fmt, _nat.stream_of(k_pages))


@torch.library.custom_op("tabicl::paged_bounds", mutates_args=("bounds", "bound_scales"))
def _paged_bounds(k_pages: Tensor, table: Tensor, lengths: Tensor, bounds: Tensor, bound_scales: Tensor,
                  start: Optional[Tensor], rows: int, scales: Optional[Tensor]) -> None:
    """See paged_bounds."""
    _bounds_launch(k_pages, table, lengths, bounds, bound_scales, start, rows, scales)


@_paged_bounds.register_fake
def _(k_pages, table, lengths, bounds, bound_scales, start, rows, scales):  # noqa: ANN001
    return None


def paged_bounds(k_pages: Tensor, table: Tensor, lengths: Tensor, bounds: Tensor, bound_scales: Tensor,
                 start: Optional[Tensor] = None, rows: Optional[int] = None, scales: Optional[Tensor] = None) -> None:
    """Writes bounds and bound_scales of the pages that hold the first lengths[n] rows of each sequence, over those rows
    of k_pages (with scales: a pool of 8-bit codes). start (int32 [N]): only of the pages from row start[n] on, and at most
    `rows` rows from there (a number: what the host knows of the rows that were appended; default: to the end). Infinite keys
    count as the end of the range, NaN not at all. The pages of other sequences keep theirs."""
    rows = (1 << 40) if rows is None else int(rows)
    if rows < 0:
        raise ValueError(f"rows must not be negative, got {rows}")
    if _nat.direct(k_pages, table, lengths, bounds, bound_scales, start, scales):
        if _nat.DIRECT is None or not _nat.DIRECT.bounds(k_pages, table, lengths, bounds, bound_scales, start, rows, scales,
                                                         _nat.stream_of(k_pages)):
            _bounds_launch(k_pages, table, lengths, bounds, bound_scales, start, rows, scales)
        torch.autograd.graph.increment_version((bounds, bound_scales))
    else:
        _pool.no_grad("paged_bounds", k_pages, bound_scales, scales)
        torch.ops.tabicl.paged_bounds(k_pages, table, lengths, bounds, bound_scales, start, min(rows, 1 << 40), scales)


def _select_launch(q: Tensor, bounds: Tensor, bound_scales: Tensor, table: Tensor, lengths: Tensor, page_rows: int,
                   index: Tensor) -> None:
    t, N = _pool.table_args(table, lengths)
    dev = table.get_device()
    if bounds.dim() != 4:
        raise ValueError(f"bounds must be [pages, H, 2, D], got {tuple(bounds.shape)}")
    P, H, _, D = bounds.shape
    _check_bounds(bounds, bound_scales, P, H, D, dev)
    if q.dim() != 4 or q.shape[0] != N or q.shape[3] != D or q.shape[1] % max(1, H):
        raise ValueError(f"q must be [{N}, a multiple of {H} heads, Tq, {D}], got {tuple(q.shape)}")
    if q.get_device() != dev or lengths.get_device() != dev or index.get_device() != dev:
        raise ValueError("q, bounds, table and lengths must be on one device")
    dt = _nat.dtype_code(q.dtype)
    if _pool.elsewhere(dev, q):
        with torch.cuda.device(dev):
            return _select_launch(q, bounds, bound_scales, table, lengths, page_rows, index)
    _, Hq, Tq, _ = q.shape
    q, qn, qh, qr = _pool.rows16(q, q.element_size())
    ws, ptr, nbytes = _pool.workspace(int(_nat.load().tabicl_paged_select_workspace_bytes(N, H, Tq, t[2])), "tabicl_paged_select", q)
    _nat.call("tabicl_paged_select", q.data_ptr(), bounds.data_ptr(), bound_scales.data_ptr(), P, page_rows, *t, lengths.data_ptr(),
              index.data_ptr(), index.shape[3], N, Hq, H, Tq, D, qn, qh, qr, dt, ptr, nbytes, _nat.stream_of(q))


def _select(q: Tensor, bounds: Tensor, bound_scales: Tensor, table: Tensor, lengths: Tensor, page_rows: int,
            pages: int) -> Tensor:
    if q.dim() != 4 or bounds.dim() != 4:
        raise ValueError(f"paged_select needs q [N, Hq, Tq, D] and bounds [pages, H, 2, D], got {tuple(q.shape)} and "
                         f"{tuple(bounds.shape)}")
    index = torch.empty(q.shape[0], bounds.shape[1], q.shape[2], pages, dtype=torch.int32, device=q.device)
    _select_launch(q, bounds, bound_scales, table, lengths, page_rows, index)
    return index


@torch.library.custom_op("tabicl::paged_select", mutates_args=())
def _paged_select(q: Tensor, bounds: Tensor, bound_scales: Tensor, table: Tensor, lengths: Tensor, page_rows: int,
                  pages: int) -> Tensor:
    """See paged_select."""
    return _select(q, bounds, bound_scales, table, lengths, page_rows, pages)


@_paged_select.register_fake
def _(q, bounds, bound_scales, table, lengths, page_rows, pages):  # noqa: ANN001
    return q.new_empty((q.shape[0], bounds.shape[1], q.shape[2], pages), dtype=torch.int32)


def paged_select(q: Tensor, bounds: Tensor, bound_scales: Tensor, table: Tensor, lengths: Tensor, page_rows: int,
                 pages: int) -> Tensor:
    """The `pages` pages of largest bound for each query row of q [N, Hq, Tq, D] (bf16 or fp32) and K/V head, as their places
    in the sequence's row of the table: int32 [N, H, Tq, pages], ascending, -1 behind the last (a sequence of fewer
    pages). Ties go to the lower page; pages that the pool has not got are not chosen. bounds, bound_scales: paged_bounds'.
    The query heads of a group choose together, by the largest of their bounds. At most 2^21 query rows over all sequences and K/V
    heads. No gradient."""
    if pages < 0:
        raise ValueError(f"pages must not be negative, got {pages}")
    if _nat.direct(q, bounds, bound_scales, table, lengths):
        if _nat.DIRECT is not None:
            index = _nat.DIRECT.select(q, bounds, bound_scales, table, lengths, int(page_rows), int(pages), _nat.stream_of(q))
            if index is not None:
                return index
        return _select(q, bounds, bound_scales, table, lengths, int(page_rows), int(pages))
    _pool.no_grad("paged_select", q, bound_scales)
    return torch.ops.tabicl.paged_select(q, bounds, bound_scales, table, lengths, int(page_rows), int(pages))


def _sparse_launch(q: Tensor, k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, index: Tensor, scale: float,
                   scales: Optional[Tensor], out: Tensor) -> None:
    pool, H, D, N, dev = _pool.pool_args(k_pages, v_pages, table, lengths)
    fmt = _pool.pool_format(k_pages, scales, dev)
    o = _pool.query_args(q, out, N, H, D, dev)
    if fmt < 2 and q.dtype is not k_pages.dtype:
        raise ValueError("q must have the pool's dtype (cast q to the cache dtype first)")
    _, Hq, Tq, _ = q.shape
    if index.dtype is not torch.int32 or index.dim() != 4 or index.shape[:3] != (N, H, Tq) or not index.is_contiguous() \
            or index.get_device() != dev:
        raise ValueError(f"index must be a contiguous int32 [{N}, {H}, {Tq}, pages] tensor on the pool's device, got {index.dtype} "
                         f"{tuple(index.shape)}")
    dt = _nat.dtype_code(q.dtype)
    if _pool.elsewhere(dev, q):
        with torch.cuda.device(dev):
            return _sparse_launch(q, k_pages, v_pages, table, lengths, index, scale, scales, out)
    q, qn, qh, qr = _pool.rows16(q, q.element_size())
    K = index.shape[3]
    ws, ptr, nbytes = _pool.workspace(int(_nat.load().tabicl_paged_sparse_attn_workspace_bytes(N, Hq, H, Tq, D, K * pool[2])),
                                      "tabicl_paged_sparse_attn", q)
    _nat.call("tabicl_paged_sparse_attn", q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
              None if scales is None else scales.data_ptr(), *pool, lengths.data_ptr(), index.data_ptr(), K, out.data_ptr(), N, Hq,
              H, Tq, D, qn, qh, qr, *o, scale, dt, fmt, ptr, nbytes, _nat.stream_of(q))


@torch.library.custom_op("tabicl::paged_sparse_attn", mutates_args=())
def _paged_sparse_attn(q: Tensor, k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, index: Tensor, scale: float,
                       scales: Optional[Tensor]) -> Tensor:
    """See paged_sparse_attention."""
    out = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    _sparse_launch(q, k_pages, v_pages, table, lengths, index, scale, scales, out)
    return out


@_paged_sparse_attn.register_fake
def _(q, k_pages, v_pages, table, lengths, index, scale, scales):  # noqa: ANN001
    return q.new_empty(q.shape)


@torch.library.custom_op("tabicl::paged_sparse_attn_out", mutates_args=("out",))
def _paged_sparse_attn_out(q: Tensor, k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, index: Tensor,
                           scale: float, scales: Optional[Tensor], out: Tensor) -> None:
    """tabicl::paged_sparse_attn written into `out`, any [N, Hq, Tq, D] view with a contiguous last dim."""
    _sparse_launch(_pool.apart(q, out), k_pages, v_pages, table, lengths, index, scale, scales, out)


@_paged_sparse_attn_out.register_fake
def _(q, k_pages, v_pages, table, lengths, index, scale, scales, out):  # noqa: ANN001
    return None


def paged_sparse_attention(q: Tensor, k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, index: Tensor,
                           scale: Optional[float] = None, out: Optional[Tensor] = None,
                           scales: Optional[Tensor] = None) -> Tensor:
    """tabicl_mi355_paged.paged_attention of each query row and K/V head over the pages that index [N, H, Tq, pages] lists
    (paged_select's, or any other: places in the table in any order, entries outside of it are skipped, a page listed
    twice counts twice). Rows past a sequence's length, and pages that the pool has not got, hold nothing; a query row
    without a row to attend to is 0. Every query row reads its own pages: for one query row to a few dozen (at most 2^22
    over all sequences and query heads). No gradient."""
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    if _nat.direct(q, k_pages, v_pages, table, lengths, index, out, scales):
        if _nat.DIRECT is not None:
            o = _nat.DIRECT.attn(q, k_pages, v_pages, scales, table, lengths, out, index, scale, _nat.stream_of(q))
            if o is not None:
                if out is not None:
                    torch.autograd.graph.increment_version(out)
                return o
        o = torch.empty_like(q, memory_format=torch.contiguous_format) if out is None else out
        _sparse_launch(q if out is None else _pool.apart(q, out), k_pages, v_pages, table, lengths, index, scale, scales, o)
        if out is not None:
            torch.autograd.graph.increment_version(out)
        return o
    _pool.no_grad("paged_sparse_attention", q, k_pages, v_pages, scales, out)
    if out is None:
        return torch.ops.tabicl.paged_sparse_attn(q, k_pages, v_pages, table, lengths, index, scale, scales)
    torch.ops.tabicl.paged_sparse_attn_out(q, k_pages, v_pages, table, lengths, index, scale, scales, out)
    return out
