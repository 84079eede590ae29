"""The paged K/V cache in 8 bits on MI355X: pools of e4m3 or int8 codes [pages, H, page_rows, D] with scales fp32
[pages, H, 2], one for K and one for V of each page and head; value = code * scale. tabicl_mi355_paged's functions come here
when they are given scales (ops tabicl::paged_attn_q8, paged_attn_q8_out, paged_append_q8, paged_gather_q8).

A scale is a power of two, the smallest 2^k (k in [-60, 100]) with max |x| <= Q 2^k, Q = 448 (e4m3) or 127 (int8). Rows that
join a page of smaller scale raise it, and the codes that the page holds are rounded to the new step: at most once per
doubling. Values are bf16 numbers, so a gather in bf16 is exact. e4m3 keeps four significant bits of each value, int8 seven
of the largest value of a page and head (a power of two as the scale may leave one of them unused), which is more for values of one
size: outputs over 5,000 normal rows are off by 3 to 8 % of their size in e4m3 and 1.4 to 2.7 % in int8, by as much and 9 to 35 %
where every sixteenth dim is 16 times as large. No counterpart in the reference."""
from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor

import tabicl_mi355_native as _nat
import tabicl_mi355_pool as _pool


def _attn_launch(q: Tensor, k_pages: Tensor, v_pages: Tensor, scales: Tensor, table: Tensor, lengths: Tensor, scale: float,
                 out: Tensor) -> None:
    pool, H, D, N, dev = _pool.pool_args(k_pages, v_pages, table, lengths)
    code = _pool.pool_format(k_pages, scales, dev) - 2
    o = _pool.query_args(q, out, N, H, D, dev)
    dt = _nat.dtype_code(q.dtype)
    if _pool.elsewhere(dev, q):
        with torch.cuda.device(dev):
            return _attn_launch(q, k_pages, v_pages, scales, table, lengths, scale, out)
    _, Hq, Tq, _ = q.shape
    q, qn, qh, qr = _pool.rows16(q, q.element_size())
    ws, ptr, nbytes = _pool.workspace(int(_nat.load().tabicl_paged_attn_q8_workspace_bytes(
        N, Hq, H, Tq, D, pool[5] * pool[2], dt)), "tabicl_paged_attn_q8", q)
    _nat.call("tabicl_paged_attn_q8", q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), scales.data_ptr(), *pool,
              lengths.data_ptr(), out.data_ptr(), N, Hq, H, Tq, D, qn, qh, qr, *o, scale, dt, code, ptr, nbytes,
              _nat.stream_of(q))


@torch.library.custom_op("tabicl::paged_attn_q8", mutates_args=())
def _paged_attn_q8(q: Tensor, k_pages: Tensor, v_pages: Tensor, scales: Tensor, table: Tensor, lengths: Tensor,
                   scale: float) -> Tensor:
    """See tabicl_mi355_paged.paged_attention."""
    out = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    _attn_launch(q, k_pages, v_pages, scales, table, lengths, scale, out)
    return out


@_paged_attn_q8.register_fake
def _(q, k_pages, v_pages, scales, table, lengths, scale):  # noqa: ANN001
    return q.new_empty(q.shape)


@torch.library.custom_op("tabicl::paged_attn_q8_out", mutates_args=("out",))
def _paged_attn_q8_out(q: Tensor, k_pages: Tensor, v_pages: Tensor, scales: Tensor, table: Tensor, lengths: Tensor,
                       scale: float, out: Tensor) -> None:
    """tabicl::paged_attn_q8 written into `out`, any [N, Hq, Tq, D] view with a contiguous last dim."""
    _attn_launch(_pool.apart(q, out), k_pages, v_pages, scales, table, lengths, scale, out)


@_paged_attn_q8_out.register_fake
def _(q, k_pages, v_pages, scales, table, lengths, scale, out):  # noqa: ANN001
    return None


def attention(q: Tensor, k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, weights: Optional[Tensor],
              scale: Optional[float], out: Optional[Tensor], scales: Tensor) -> Tensor:
    """tabicl_mi355_paged.paged_attention of a pool of 8-bit codes."""
    if weights is not None:
        raise ValueError("paged_attention over 8-bit codes adds up no weights")
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    if _nat.direct(q, k_pages, v_pages, scales, table, lengths, out):
        if _nat.DIRECT is not None:
            o = _nat.DIRECT.attn(q, k_pages, v_pages, scales, table, lengths, out, None, scale, _nat.stream_of(q))
            if o is not None:
                if out is not None:
                    torch.autograd.graph.increment_version(out)
                return o
        o = torch.empty_like(q, memory_format=torch.contiguous_format) if out is None else out
        _attn_launch(q if out is None else _pool.apart(q, out), k_pages, v_pages, scales, table, lengths, scale, o)
        if out is not None:
            torch.autograd.graph.increment_version(out)
        return o
    _pool.no_grad("paged_attention", q, k_pages, v_pages, scales, out)
    if out is None:
        return torch.ops.tabicl.paged_attn_q8(q, k_pages, v_pages, scales, table, lengths, scale)
    torch.ops.tabicl.paged_attn_q8_out(q, k_pages, v_pages, scales, table, lengths, scale, out)
    return out


def _append_launch(k_pages: Tensor, v_pages: Tensor, scales: Tensor, table: Tensor, lengths: Tensor, k: Tensor, v: Tensor,
                   count: Optional[Tensor], starts: Optional[Tensor]) -> None:
    pool, H, D, N, dev = _pool.pool_args(k_pages, v_pages, table, lengths)
    code = _pool.pool_format(k_pages, scales, dev) - 2
    packed = starts is not None
    shape = k.shape
    want = (k.shape[0], H, D) if packed else (N, H, k.shape[2] if k.dim() == 4 else 0, D)
    if k.dim() != len(want) or v.shape != shape or shape != want:
        raise ValueError(f"k and v must be [{'total' if packed else N}, {H}{'' if packed else ', T'}, {D}], got {tuple(shape)} and "
                         f"{tuple(v.shape)}")
    dt = _nat.dtype_code(k.dtype)
    if v.dtype is not k.dtype:
        raise ValueError("k and v must share a dtype")
    if packed:
        _pool.counts(starts, N + 1, "starts")
    if count is not None:
        _pool.counts(count, N, "count")
    if any(t is not None and t.get_device() != dev for t in (k, v, count, starts)):
        raise ValueError("k, v, count, starts and the pool must be on one device")
    if _pool.elsewhere(dev, k):
        with torch.cuda.device(dev):
            return _append_launch(k_pages, v_pages, scales, table, lengths, k, v, count, starts)
    es = k.element_size()
    if packed:  # [total, H, D] as [1, H, total, D]
        k, v = k.unsqueeze(0).transpose(1, 2), v.unsqueeze(0).transpose(1, 2)
    k, kn, kh, kr = _pool.rows16(k, es)
    v, vn, vh, vr = _pool.rows16(v, es)
    _nat.call("tabicl_paged_append_q8", k_pages.data_ptr(), v_pages.data_ptr(), scales.data_ptr(), *pool, lengths.data_ptr(),
              k.data_ptr(), v.data_ptr(), None if count is None else count.data_ptr(), starts.data_ptr() if packed else None, N, H,
              k.shape[2], D, kn, kh, kr, vn, vh, vr, dt, code, _nat.stream_of(k))


@torch.library.custom_op("tabicl::paged_append_q8", mutates_args=("k_pages", "v_pages", "scales"))
def _paged_append_q8(k_pages: Tensor, v_pages: Tensor, scales: Tensor, table: Tensor, lengths: Tensor, k: Tensor, v: Tensor,
                     count: Optional[Tensor] = None, starts: Optional[Tensor] = None) -> None:
    """See tabicl_mi355_paged.paged_append; with starts, paged_append_packed."""
    _append_launch(k_pages, v_pages, scales, table, lengths, k, v, count, starts)


@_paged_append_q8.register_fake
def _(k_pages, v_pages, scales, table, lengths, k, v, count=None, starts=None):  # noqa: ANN001
    return None


def append(k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, k: Tensor, v: Tensor, count: Optional[Tensor],
           starts: Optional[Tensor], scales: Optional[Tensor]) -> None:
    """tabicl_mi355_paged.paged_append (or, with starts, paged_append_packed) to a pool of 8-bit codes."""
    if scales is None:
        raise ValueError("a pool of 8-bit codes needs its scales [pages, H, 2]")
    if _nat.direct(k_pages, v_pages, scales, table, lengths, k, v, count, starts):
        if starts is not None or _nat.DIRECT is None or not _nat.DIRECT.append(k_pages, v_pages, scales, table, lengths, k, v, count,
                                                                               _nat.stream_of(k)):
            _append_launch(k_pages, v_pages, scales, table, lengths, k, v, count, starts)
        torch.autograd.graph.increment_version((k_pages, v_pages, scales))
    else:
        _pool.no_grad("paged_append", k_pages, v_pages, scales, k, v)
        torch.ops.tabicl.paged_append_q8(k_pages, v_pages, scales, table, lengths, k, v, count, starts)


def _gather_launch(k_pages: Tensor, v_pages: Tensor, scales: Tensor, table: Tensor, lengths: Tensor, k: Tensor,
                   v: Tensor) -> None:
    pool, H, D, N, dev = _pool.pool_args(k_pages, v_pages, table, lengths)
    code = _pool.pool_format(k_pages, scales, dev) - 2
    if _pool.elsewhere(dev, k_pages):
        with torch.cuda.device(dev):
            return _gather_launch(k_pages, v_pages, scales, table, lengths, k, v)
    _nat.call("tabicl_paged_gather_q8", k_pages.data_ptr(), v_pages.data_ptr(), scales.data_ptr(), *pool, lengths.data_ptr(),
              k.data_ptr(), v.data_ptr(), N, H, k.shape[2], D, _nat.dtype_code(k.dtype), code, _nat.stream_of(k_pages))


def _gather(k_pages: Tensor, v_pages: Tensor, scales: Tensor, table: Tensor, lengths: Tensor, rows: int,
            dtype: torch.dtype) -> tuple[Tensor, Tensor]:
    shape = (table.shape[0], k_pages.shape[1], rows, k_pages.shape[3])
    k = torch.empty(shape, dtype=dtype, device=k_pages.device)
    v = torch.empty_like(k)
    _gather_launch(k_pages, v_pages, scales, table, lengths, k, v)
    return k, v


@torch.library.custom_op("tabicl::paged_gather_q8", mutates_args=())
def _paged_gather_q8(k_pages: Tensor, v_pages: Tensor, scales: Tensor, table: Tensor, lengths: Tensor, rows: int,
                     dtype: torch.dtype) -> tuple[Tensor, Tensor]:
    """See tabicl_mi355_paged.paged_gather."""
    return _gather(k_pages, v_pages, scales, table, lengths, rows, dtype)


@_paged_gather_q8.register_fake
def _(k_pages, v_pages, scales, table, lengths, rows, dtype):  # noqa: ANN001
    shape = (table.shape[0], k_pages.shape[1], rows, k_pages.shape[3])
    return k_pages.new_empty(shape, dtype=dtype), v_pages.new_empty(shape, dtype=dtype)


def gather(k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, rows: int, scales: Optional[Tensor],
           dtype: Optional[torch.dtype]) -> tuple[Tensor, Tensor]:
    """tabicl_mi355_paged.paged_gather of a pool of 8-bit codes."""
    if scales is None:
        raise ValueError("a pool of 8-bit codes needs its scales [pages, H, 2]")
    dtype = torch.bfloat16 if dtype is None else dtype
    _nat.dtype_code(dtype)
    if _nat.direct(k_pages, v_pages, scales, table, lengths):
        if _nat.DIRECT is not None:
            kv = _nat.DIRECT.gather(k_pages, v_pages, scales, table, lengths, rows, dtype is torch.float32, _nat.stream_of(k_pages))
            if kv is not None:
                return kv
        return _gather(k_pages, v_pages, scales, table, lengths, rows, dtype)
    _pool.no_grad("paged_gather", k_pages, v_pages, scales)
    return torch.ops.tabicl.paged_gather_q8(k_pages, v_pages, scales, table, lengths, rows, dtype)
