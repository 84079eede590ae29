"""A paged K/V cache of the ICL stage on MI355X: tables of different sizes share one pool of pages, a test row or a few
attend over the cached train rows of their table, and a cache over its budget keeps the rows the queries attended to.

IclKVCache (tabicl_mi355_icl.py) gives every estimator of a cache the same capacity; a service that holds many tables at
once, that gets its train rows over time or answers one test row at a time keeps them here instead:
  * paged_attention(q, k_pages, v_pages, table, lengths, weights) (ops tabicl::paged_attn, paged_attn_out,
    paged_attn_weights_out): attention of few query rows over the cached rows, optionally adding up the attention weight
    that each cached row drew;
  * paged_append, paged_gather (ops of these names): new rows into the pages, rows out of them;
  * paged_evict (op tabicl::paged_evict_out): cuts sequences to their rows of largest weight, in place;
  * the same over pools of 8-bit codes, with `scales` (tabicl_mi355_paged8); attention over selected pages: paged_bounds,
    paged_select, paged_sparse_attention (tabicl_mi355_sparse); page tables and slot maps kept on the GPU: paged_reserve,
    paged_slots, paged_append_packed, paged_release (tabicl_mi355_books);
  * PagedIclKVCache: the pool, the page table and the lengths, with the surface of IclKVCache (append, query,
    attention_layer, query_blocks, usable as cached_query's icl_cache), and evict.

A pool is [pages, H, page_rows, D] per block for K and V (bf16 or fp32, head dim 32, 64 or 128, page_rows a power of two
from 16 on): a (page, head) is page_rows contiguous rows. Row i of sequence n is row i % page_rows of page
table[n, i // page_rows]; table and lengths are int32 on the GPU and never read back, so a call can be captured in a
graph. A page id outside the pool holds no rows. The order of a sequence's rows carries no meaning (a train row's
position is not part of its key), which is what lets eviction fill the places of evicted rows with rows from the end.
No counterpart in the reference, whose cache is one padded tensor per block (scripts/tabicl_tpu_bucketed.py:413-435)."""
from __future__ import annotations

from typing import Callable, Optional, Sequence, Union

import torch
import torch.nn.functional as F
from torch import Tensor

import tabicl_mi355_icl as _icl
import tabicl_mi355_native as _nat
import tabicl_mi355_paged8 as _p8
import tabicl_mi355_pool as _pool
from tabicl_mi355_books import paged_append_packed, paged_release, paged_reserve, paged_slots  # noqa: F401
from tabicl_mi355_sparse import paged_bounds, paged_select, paged_sparse_attention  # noqa: F401


_rows16, _apart, _no_grad, _fwd_level, _pool_args = _pool.rows16, _pool.apart, _pool.no_grad, _pool.fwd_level, _pool.pool_args


def _check_weights(weights: Tensor, N: int, cap: int, dev: int) -> int:
    """The row stride of weights [N, >= cap]."""
    shape = weights.shape
    if weights.dtype is not torch.float32 or len(shape) != 2 or shape[0] != N or shape[1] < cap \
            or (shape[1] > 1 and weights.stride(1) != 1) or weights.get_device() != dev:
        raise ValueError(f"weights must be a float32 [{N}, >= {cap}] tensor with contiguous rows on the table's device, got "
                         f"{weights.dtype} {tuple(shape)}")
    return weights.stride(0) if N > 1 else shape[1]


_WS_BYTES: dict = {}


def _ws_bytes(key: tuple, N: int, Hq: int, H: int, Tq: int, D: int, rows: int, weighted: int, code: int) -> int:
    nbytes = int(_nat.load().tabicl_paged_attn_workspace_bytes(N, Hq, H, Tq, D, rows, weighted, code))
    if nbytes < 0:
        raise _nat.UnsupportedShapeError(f"tabicl_paged_attn: {_nat.last_error()}")
    if len(_WS_BYTES) >= 4096:  # lengths that grow row by row bring new keys for ever
        _WS_BYTES.clear()
    _WS_BYTES[key] = nbytes
    return nbytes


def _attn_launch(q: Tensor, k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, weights: Optional[Tensor],
                 scale: float, out: Tensor) -> None:
    pool, H, D, N, dev = _pool_args(k_pages, v_pages, table, lengths)
    code = _pool.dense_code(k_pages.dtype)
    shape = q.shape
    if len(shape) != 4 or shape[0] != N or shape[3] != D or shape[1] % max(1, H):
        raise ValueError(f"q must be [{N}, a multiple of {H} heads, Tq, {D}], got {tuple(shape)}")
    if out.shape != shape or out.dtype is not q.dtype or q.dtype is not k_pages.dtype:
        raise ValueError("out must match q, and both the pool's dtype (cast q to the cache dtype first)")
    if q.get_device() != dev or out.get_device() != dev:
        raise ValueError("q, out and the pool must be on one device")
    rows = pool[5] * pool[2]
    w_ptr = w_sn = 0
    if weights is not None:
        w_sn = _check_weights(weights, N, rows, dev)
        w_ptr = weights.data_ptr()
    if dev != torch.cuda.current_device() if dev >= 0 else True:  # a HIP launch goes by the current device
        _nat.require_device(q)
        with torch.cuda.device(dev):
            return _attn_launch(q, k_pages, v_pages, table, lengths, weights, scale, out)
    _, Hq, Tq, _ = shape
    q, qn, qh, qr = _rows16(q, q.element_size())
    on, oh, orow, od = out.stride()
    if od != 1 or (N > 1 and on == 0) or (Hq > 1 and oh == 0) or (Tq > 1 and orow == 0):
        raise ValueError("out needs a contiguous last dim and a place of its own for each row")
    on, oh, orow = on if N > 1 else 0, oh if Hq > 1 else 0, orow if Tq > 1 else 0
    key = (N, Hq, H, Tq, D, rows, w_ptr != 0, code, dev)
    nbytes = _WS_BYTES.get(key)
    if nbytes is None:
        nbytes = _ws_bytes(key, N, Hq, H, Tq, D, rows, w_ptr != 0, code)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
    _nat.call("tabicl_paged_attn", q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), *pool, lengths.data_ptr(),
              w_ptr or None, w_sn, out.data_ptr(), N, Hq, H, Tq, D, qn, qh, qr, on, oh, orow, scale, code,
              None if ws is None else ws.data_ptr(), nbytes, _nat.stream_of(q))


# Three ops, since torch.compile refuses an op that returns a tensor and may or may not change another.
@torch.library.custom_op("tabicl::paged_attn", mutates_args=())
def _paged_attn(q: Tensor, k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, scale: float) -> Tensor:
    """See paged_attention."""
    out = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    _attn_launch(q, k_pages, v_pages, table, lengths, None, scale, out)
    return out


@_paged_attn.register_fake
def _(q, k_pages, v_pages, table, lengths, scale):  # noqa: ANN001
    return q.new_empty(q.shape)


@torch.library.custom_op("tabicl::paged_attn_out", mutates_args=("out",))
def _paged_attn_out(q: Tensor, k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, scale: float,
                    out: Tensor) -> None:
    """tabicl::paged_attn written into `out`, any [N, Hq, Tq, D] view with a contiguous last dim."""
    _attn_launch(_apart(q, out), k_pages, v_pages, table, lengths, None, scale, out)


@_paged_attn_out.register_fake
def _(q, k_pages, v_pages, table, lengths, scale, out):  # noqa: ANN001
    return None


@torch.library.custom_op("tabicl::paged_attn_weights_out", mutates_args=("out", "weights"))
def _paged_attn_weights_out(q: Tensor, k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, scale: float,
                            out: Tensor, weights: Tensor) -> None:
    """tabicl::paged_attn_out that adds the attention weights to `weights` in place."""
    _attn_launch(_apart(q, out), k_pages, v_pages, table, lengths, weights, scale, out)


@_paged_attn_weights_out.register_fake
def _(q, k_pages, v_pages, table, lengths, scale, out, weights):  # noqa: ANN001
    return None


def paged_attention(q: Tensor, k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor,
                    weights: Optional[Tensor] = None, scale: Optional[float] = None, out: Optional[Tensor] = None,
                    scales: Optional[Tensor] = None) -> Tensor:
    """softmax(q k^T scale) v of q [N, Hq, Tq, D] over the first lengths[n] rows of each sequence n of a paged pool
    (k_pages, v_pages [pages, H, page_rows, D]; Hq a multiple of H, query head h reads K/V head h // (Hq // H); table
    [N, max_pages] and lengths [N] int32; scale defaults to D^-0.5). Returns [N, Hq, Tq, D] in q's dtype, the pool's;
    rows of an empty sequence, or whose every score is -inf, are 0. Scores, softmax and the value products are fp32
    sums. weights: an optional fp32 [N, >= max_pages page_rows] tensor; the probabilities of each cached row, summed over
    query heads and rows, are added to it in place (entries past the length are left as they are), always in the same
    order of sums. out: written in place of a new tensor, any [N, Hq, Tq, D] view whose last dim is contiguous and whose
    rows start on 16 bytes (q itself, too).

    The work is split over the cached rows, so one test row over one long table fills the GPU; a table slice
    table[:, :w] that covers the longest sequence spares the workgroups of pages nobody holds. For up to a few hundred
    query rows (each group of 64 reads the cache again); with weights, more go in slices where the workspace would pass
    1 GiB. No gradient.

    scales (fp32 [pages, H, 2]): the pool holds e4m3 or int8 codes (tabicl_mi355_paged8). q is bf16 or fp32 then; the products
    are exact, the sums fp32 (bf16 probabilities take part as two bf16 terms, fp32 ones as three). No weights."""
    if scales is not None:
        return _p8.attention(q, k_pages, v_pages, table, lengths, weights, scale, out, scales)
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    if _nat.direct(q, k_pages, v_pages, table, lengths, weights, out):
        o = torch.empty_like(q, memory_format=torch.contiguous_format) if out is None else out
        _attn_launch(q if out is None else _apart(q, out), k_pages, v_pages, table, lengths, weights, scale, o)
        if out is not None:
            torch.autograd.graph.increment_version(out)
        if weights is not None:
            torch.autograd.graph.increment_version(weights)
        return o
    _no_grad("paged_attention", q, k_pages, v_pages, weights, out)
    if out is None and weights is None:
        return torch.ops.tabicl.paged_attn(q, k_pages, v_pages, table, lengths, scale)
    out = q.new_empty(q.shape) if out is None else out
    if weights is None:
        torch.ops.tabicl.paged_attn_out(q, k_pages, v_pages, table, lengths, scale, out)
    else:
        torch.ops.tabicl.paged_attn_weights_out(q, k_pages, v_pages, table, lengths, scale, out, weights)
    return out


def _append_launch(k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, k: Tensor, v: Tensor,
                   count: Optional[Tensor]) -> None:
    pool, H, D, N, dev = _pool_args(k_pages, v_pages, table, lengths)
    code = _pool.dense_code(k_pages.dtype)
    shape = k.shape
    if len(shape) != 4 or v.shape != shape or shape[0] != N or shape[1] != H or shape[3] != D:
        raise ValueError(f"k and v must be [{N}, {H}, T, {D}], got {tuple(shape)} and {tuple(v.shape)}")
    if k.dtype is not k_pages.dtype or v.dtype is not k_pages.dtype:
        raise ValueError(f"paged_append expects {k_pages.dtype} (cast before appending)")
    if count is not None and (count.dtype is not torch.int32 or count.shape != (N,) or not count.is_contiguous()
                              or count.get_device() != dev):
        raise ValueError(f"count must be a contiguous int32 tensor of {N} entries on the pool's device")
    if k.get_device() != dev or v.get_device() != dev:
        raise ValueError("k, v and the pool must be on one device")
    if dev != torch.cuda.current_device() if dev >= 0 else True:
        _nat.require_device(k)
        with torch.cuda.device(dev):
            return _append_launch(k_pages, v_pages, table, lengths, k, v, count)
    es = k.element_size()
    k, kn, kh, kr = _rows16(k, es)
    v, vn, vh, vr = _rows16(v, es)
    _nat.call("tabicl_paged_append", k_pages.data_ptr(), v_pages.data_ptr(), *pool, lengths.data_ptr(), k.data_ptr(),
              v.data_ptr(), None if count is None else count.data_ptr(), N, H, shape[2], D, kn, kh, kr, vn, vh, vr, code,
              _nat.stream_of(k))


@torch.library.custom_op("tabicl::paged_append", mutates_args=("k_pages", "v_pages"))
def _paged_append(k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, k: Tensor, v: Tensor,
                  count: Optional[Tensor] = None) -> None:
    """See paged_append."""
    _append_launch(k_pages, v_pages, table, lengths, k, v, count)


@_paged_append.register_fake
def _(k_pages, v_pages, table, lengths, k, v, count=None):  # noqa: ANN001
    return None


def paged_append(k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, k: Tensor, v: Tensor,
                 count: Optional[Tensor] = None, scales: Optional[Tensor] = None) -> None:
    """Rows t < count[n] (int32 [N]; default all) of k, v [N, H, T, D] into rows lengths[n] + t of each sequence of the
    pool (any strides with a contiguous last dim, e.g. the heads of a K|V projection). lengths is read, not changed: the
    other blocks of a model append at the same rows. Rows that the table has no page for are dropped. A page that
    is written must stand in the table once.

    scales (fp32 [pages, H, 2], written too): the pool holds e4m3 or int8 codes; k and v are bf16 or fp32. A page that rows
    join keeps the larger of its scale and theirs, and the codes it holds are rounded again where it grows; infinities saturate,
    NaN stays NaN in e4m3 and becomes 0 in int8."""
    if scales is not None:
        _p8.append(k_pages, v_pages, table, lengths, k, v, count, None, scales)
    elif _nat.direct(k_pages, v_pages, table, lengths, k, v, count):
        _append_launch(k_pages, v_pages, table, lengths, k, v, count)
        torch.autograd.graph.increment_version((k_pages, v_pages))
    else:
        _no_grad("paged_append", k_pages, v_pages, k, v)
        torch.ops.tabicl.paged_append(k_pages, v_pages, table, lengths, k, v, count)


def _gather_launch(k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, k: Tensor, v: Tensor) -> None:
    pool, H, D, N, dev = _pool_args(k_pages, v_pages, table, lengths)
    code = _pool.dense_code(k_pages.dtype)
    if dev != torch.cuda.current_device() if dev >= 0 else True:
        _nat.require_device(k_pages)
        with torch.cuda.device(dev):
            return _gather_launch(k_pages, v_pages, table, lengths, k, v)
    _nat.call("tabicl_paged_gather", k_pages.data_ptr(), v_pages.data_ptr(), *pool, lengths.data_ptr(), k.data_ptr(),
              v.data_ptr(), N, H, k.shape[2], D, code, _nat.stream_of(k))


def _gather(k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, rows: int) -> tuple[Tensor, Tensor]:
    shape = (table.shape[0], k_pages.shape[1], rows, k_pages.shape[3])
    k, v = k_pages.new_empty(shape), v_pages.new_empty(shape)
    _gather_launch(k_pages, v_pages, table, lengths, k, v)
    return k, v


@torch.library.custom_op("tabicl::paged_gather", mutates_args=())
def _paged_gather(k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, rows: int) -> tuple[Tensor, Tensor]:
    """See paged_gather."""
    return _gather(k_pages, v_pages, table, lengths, rows)


@_paged_gather.register_fake
def _(k_pages, v_pages, table, lengths, rows):  # noqa: ANN001
    shape = (table.shape[0], k_pages.shape[1], rows, k_pages.shape[3])
    return k_pages.new_empty(shape), v_pages.new_empty(shape)


def paged_gather(k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, rows: int, scales: Optional[Tensor] = None,
                 dtype: Optional[torch.dtype] = None) -> tuple[Tensor, Tensor]:
    """k, v [N, H, rows, D] with the first min(lengths[n], rows) rows of each sequence side by side, 0 where a row has no
    page; what lies past a sequence's length is not written. For calls that the dense kernels answer faster (many query
    rows), or to copy a cache out of its pool. In the pool's dtype; with scales (a pool of e4m3 or int8 codes) the values in
    `dtype`, bf16 (the default: they are bf16 numbers) or fp32."""
    if k_pages.dim() != 4 or rows < 0:
        raise ValueError(f"paged_gather needs pools [pages, H, page_rows, D] and rows >= 0, got {tuple(k_pages.shape)}, {rows}")
    if scales is not None or k_pages.dtype in _pool.CODES:
        return _p8.gather(k_pages, v_pages, table, lengths, int(rows), scales, dtype)
    _no_grad("paged_gather", k_pages, v_pages)
    if dtype is not None and dtype is not k_pages.dtype:
        raise ValueError(f"a {k_pages.dtype} pool is gathered in its own dtype")
    if _nat.direct(k_pages, v_pages, table, lengths):
        return _gather(k_pages, v_pages, table, lengths, int(rows))
    return torch.ops.tabicl.paged_gather(k_pages, v_pages, table, lengths, int(rows))


def _evict_launch(k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, weights: Tensor, keep: int,
                  recent: int, keep_n: Optional[Tensor], index: Tensor, kept_weights: Tensor, kept: Tensor) -> None:
    pool, H, D, N, dev = _pool_args(k_pages, v_pages, table, lengths, 1)
    code = _nat.dtype_code(k_pages.dtype)
    w_sn = _check_weights(weights, N, pool[2] * pool[5], dev)
    if keep < 0 or recent < 0:
        raise ValueError(f"keep and recent must not be negative, got {keep} and {recent}")
    if keep_n is not None and (keep_n.dtype is not torch.int32 or keep_n.shape != (N,) or not keep_n.is_contiguous()
                               or keep_n.get_device() != dev):
        raise ValueError(f"keep must be a number or a contiguous int32 tensor of {N} entries on the table's device")
    if dev != torch.cuda.current_device() if dev >= 0 else True:
        _nat.require_device(table)
        with torch.cuda.device(dev):
            return _evict_launch(k_pages, v_pages, table, lengths, weights, keep, recent, keep_n, index, kept_weights, kept)
    B, cap = k_pages.shape[0], pool[2] * pool[5]
    K = min(keep, cap)
    nbytes = int(_nat.load().tabicl_paged_evict_workspace_bytes(N, K))  # not kept: K changes with the data
    if nbytes < 0:
        raise _nat.UnsupportedShapeError(f"tabicl_paged_evict: {_nat.last_error()}")
    ws = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=table.device)
    _nat.call("tabicl_paged_evict", k_pages.data_ptr(), v_pages.data_ptr(), B, k_pages.stride(0) if B > 1 else 0, *pool,
              lengths.data_ptr(), weights.data_ptr(), w_sn, None if keep_n is None else keep_n.data_ptr(), keep, recent,
              index.data_ptr(), K, kept_weights.data_ptr(), kept.data_ptr(), N, H, D, code, ws.data_ptr(), nbytes,
              _nat.stream_of(table))


@torch.library.custom_op("tabicl::paged_evict_out", mutates_args=("k_pages", "v_pages", "index", "kept_weights", "kept"))
def _paged_evict_out(k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, weights: Tensor, keep: int,
                     recent: int, keep_n: Optional[Tensor], index: Tensor, kept_weights: Tensor, kept: Tensor) -> None:
    """See paged_evict; keep_n is its tensor keep (keep then bounds it)."""
    N, cap = table.shape[0], table.shape[1] * k_pages.shape[-2]
    for t, shape, dtype in ((index, (N, max(0, min(keep, cap))), torch.int32), (kept_weights, (N, cap), torch.float32),
                            (kept, (N,), torch.int32)):
        if t.shape != shape or t.dtype is not dtype or not t.is_contiguous() or t.device != table.device:
            raise ValueError(f"eviction writes to contiguous {dtype} {shape}, got {t.dtype} {tuple(t.shape)}")
    _evict_launch(k_pages, v_pages, table, lengths, weights, keep, recent, keep_n, index, kept_weights, kept)


@_paged_evict_out.register_fake
def _(k_pages, v_pages, table, lengths, weights, keep, recent, keep_n, index, kept_weights, kept):  # noqa: ANN001
    return None


def paged_evict(k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, weights: Tensor,
                keep: Union[int, Tensor], recent: int = 0) -> tuple[Tensor, Tensor, Tensor]:
    """Cuts each sequence to kept = min(lengths[n], keep) rows (keep: a number, or int32 [N] on the GPU) in all blocks of
    k_pages, v_pages [blocks, pages, H, page_rows, D] (or one block [pages, H, page_rows, D]), in place. Kept are its last
    min(recent, kept) rows and, of those before them, the rows of the largest weights [N, >= max_pages page_rows] (fp32;
    ties: the lower row; NaN counts as -inf). Kept rows past the cut move, in order, to the places of the evicted ones
    below it; nothing else moves. Returns index [N, K] int32 (slot j holds the old row index[n, j], -1 from kept on; K =
    keep, or the capacity for a tensor), the weights in their new slots [N, max_pages page_rows] (0 past the cut) and
    kept [N] int32. weights, table and lengths are not changed: take over the new ones. No page may stand in the table
    twice. A row below the length whose page the pool does not have is ranked by its weight like any other; a kept row whose
    new place has no page is nowhere afterwards."""
    if k_pages.dim() == 4 and v_pages.dim() == 4:
        k_pages, v_pages = k_pages.unsqueeze(0), v_pages.unsqueeze(0)
    keep_n = None
    N, cap = table.shape[0], table.shape[1] * k_pages.shape[3] if k_pages.dim() == 5 else 0
    if isinstance(keep, Tensor):
        keep, keep_n = cap, keep
    keep, recent = min(int(keep), cap), min(int(recent), cap)  # the entry points take 64 bits
    index = table.new_empty(N, max(0, min(keep, cap)))
    kept_weights = weights.new_empty(N, cap)
    kept = table.new_empty(N)
    if _nat.direct(k_pages, v_pages, table, lengths, weights, keep_n):
        _evict_launch(k_pages, v_pages, table, lengths, weights, keep, recent, keep_n, index, kept_weights, kept)
        torch.autograd.graph.increment_version((k_pages, v_pages))
    else:
        _no_grad("paged_evict", k_pages, v_pages, weights)
        torch.ops.tabicl.paged_evict_out(k_pages, v_pages, table, lengths, weights, keep, recent, keep_n, index, kept_weights,
                                         kept)
    return index, kept_weights, kept


# PagedIclKVCache.query gathers a block's rows for the dense kernel, which shares each tile of K and V among 256 query rows,
# from so many query rows, so many of them over all sequences (it has too few tiles for the GPU below) and so many products of
# query rows and cached rows (per head) on. us in the pages / gathered, for query rows T:
#   8 x 45,000 cached rows T 192 419 / 450, 256 443 / 462, 257 644 / 549, 1000 1641 / 899; 40 x 100 to 20,000 256 641 / 571;
#   8 x 5,000 256 68 / 64, 512 114 / 81; 8 x 20,000 256 208 / 207, 320 254 / 266, 384 299 / 265; 8 x 700 512 39 / 56,
#   5000 285 / 88;
#   1 x 45,000 384 87 / 186, 1000 184 / 192, 1500 266 / 194; 2 x 45,000 384 146 / 216, 512 184 / 217, 700 300 / 219;
#   4 x 45,000 256 181 / 279, 384 281 / 304, 512 352 / 311; 1 x 200,000 700 674 / 808, 1000 804 / 797.
_DENSE_QUERY_ROWS, _DENSE_ALL_ROWS, _DENSE_SCORES = 256, 1024, 1 << 24
# Bytes of K and V that a gather puts side by side (more only for a single sequence of more): the sequences go in runs, each
# padded to its own longest one. us of all at once / in runs of 2 GiB / 1 GiB, T 384: 16 x 45,000 rows 1246 / 1243 / 1262, one
# table of 50,000 rows beside 63 of 500 752 (6.3 GB) / 514 / 507, 40 of 100 to 20,000 763 / 713 / 829.
_GATHER_BYTES = 2 << 30
# What paged_select (query rows over sequences and K/V heads) and paged_sparse_attention (over sequences and query heads) take in a
# call, and the bytes of the list of pages and of selection's workspace that a query over selected pages keeps at a time.
_SELECT_ROWS, _SPARSE_ROWS, _SELECT_BYTES = 1 << 21, 1 << 22, 1 << 30


class PagedIclKVCache(_icl.IclKVCache):
    """The ICL stage's K/V cache in pages: `sequences` (tables, or estimators of tables) of up to max_rows rows each, in
    `pages` pages of page_rows rows that every block holds one of ([blocks, pages, heads, page_rows, head_dim] for K and
    V). append, append_projected, query, attention_layer, query_blocks and query_chunked as in IclKVCache (rows go behind
    each sequence's last one, and a sequence may get fewer rows than the others of a call); cached_query takes it as its
    icl_cache.

    track=True adds up, over every query of every block, the attention weight that each cached row draws (`weights`, fp32
    [sequences, capacity]); evict(keep) cuts the sequences to their heaviest rows and returns the emptied pages.

    dtype torch.float8_e4m3fn or torch.int8: rows are held in 8 bits with a scale for each page and head (`scales`, fp32 [blocks,
    pages, heads, 2]; tabicl_mi355_paged8), appended in bf16 or fp32 and queried in either. Not with track.

    select=K: each query row of each head attends to the K pages of its table whose keys can give it the largest scores
    (tabicl_mi355_sparse; all of them, where a table has no more), however many rows a query has (they go in slices). The bounds of the keys
    (`bounds`, `bound_scales`) follow the appends. Not with track. Each query row and head reads its own pages, which is faster than all
    pages for few rows over many pages alone (us of all / 64 pages of 64 rows, 8 x 45,000 rows of 64 dims in bf16: one row 131 / 33, 16
    rows 133 / 126, 32 rows 135 / 209, 1,000 rows 938 / 5,708; 8 x 5,000 rows, one row 26 / 32).

    Pages are given out on the host; the page table and the lengths live on the GPU, so a query costs no host sync. Calls
    follow each other on one stream. Only queries can be captured in a graph and replayed as the cache grows (the other calls
    keep books on the host)."""

    def __init__(self, sequences: int, blocks: int, heads: int, head_dim: int, max_rows: int, pages: int,
                 page_rows: int = 64, dtype: torch.dtype = torch.bfloat16, device: Union[str, torch.device] = "cuda",
                 track: bool = False, select: Optional[int] = None):
        q8 = dtype in _pool.CODES
        if track and (q8 or select is not None):
            raise ValueError("a cache of 8-bit rows, or one whose queries select pages, tracks no weights")
        if select is not None and select < 1:
            raise ValueError(f"select must be at least 1, got {select}")
        if page_rows < 16 or page_rows & (page_rows - 1):
            raise ValueError(f"page_rows must be a power of two from 16 on, got {page_rows}")
        width = -(-max_rows // page_rows)
        with torch.inference_mode(False):  # tensors that calls in and outside of inference mode may change
            self.keys = torch.empty(blocks, pages, heads, page_rows, head_dim, dtype=dtype, device=device)
            self.values = torch.empty_like(self.keys)
            self.table = torch.full((sequences, width), -1, dtype=torch.int32, device=device)
            self.lengths = torch.zeros(blocks, sequences, dtype=torch.int32, device=device)
            self.weights = torch.zeros(sequences, width * page_rows, dtype=torch.float32, device=device) if track else None
            self._pages = torch.full((sequences, width), -1, dtype=torch.int32)  # the table's host copy
            self.scales = torch.zeros(blocks, pages, heads, 2, dtype=torch.float32, device=device) if q8 else None
            self.bounds = self.bound_scales = None
            if select is not None:
                self.bounds = torch.zeros(blocks, pages, heads, 2, head_dim, dtype=torch.int8, device=device)
                self.bound_scales = torch.zeros(blocks, pages, heads, dtype=torch.float32, device=device)
        self.select = select
        self.page_rows = page_rows
        self.capacity = width * page_rows
        self._held = [0] * sequences  # pages a sequence holds
        self._rows = [[0] * sequences for _ in range(blocks)]  # the lengths' host copy
        self._free = list(range(pages - 1, -1, -1))
        self._root, self._first = self, 0  # of a view: the cache it shows, and its first sequence there

    @property
    def shape(self):
        """(sequences, blocks, heads, capacity, head_dim), as of IclKVCache."""
        B, _, H, _, D = self.keys.shape
        return (self.table.shape[0], B, H, self.capacity, D)

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _lengths_of(self, block: int) -> list:
        """The block's lengths on the host (of a view: as the cache it shows has them now)."""
        return self._root._rows[block][self._first:self._first + self.table.shape[0]]

    def length(self, block: int, sequence: int = 0) -> int:
        return self._lengths_of(block)[sequence]

    def default_valid(self, block: int) -> Tensor:
        """The block's filled lengths as the int32 device tensor the kernels take (of a view too: a table without rows
        answers 0 as long as another one of the cache it shows has some)."""
        if not any(self._root._rows[block]):
            raise ValueError(f"block {block} of the cache has no rows: append before querying")
        return self.lengths[block]

    def _capturing(self) -> bool:
        return self.keys.is_cuda and torch.cuda.is_current_stream_capturing()

    def _own(self, what: str) -> None:
        if self._root is not self:
            raise ValueError(f"{what}: a view of some of a cache's estimators answers queries only")
        if self._capturing():  # a replay would repeat what it did on the GPU and not what it wrote down here
            raise ValueError(f"{what} keeps books on the host: only queries can be captured in a graph")

    def reserve(self, rows: Union[int, Sequence[int]]) -> None:
        """Pages for sequences of up to `rows` rows (a number, or one per sequence), given out now rather than by the
        appends that fill them. They stay a sequence's own until it is released or the cache evicts."""
        self._own("reserve")
        S, R = self.table.shape[0], self.page_rows
        rows = [int(rows)] * S if isinstance(rows, int) else [int(r) for r in rows]
        if len(rows) != S:
            raise ValueError(f"{len(rows)} row counts for {S} sequences")
        if max(rows, default=0) > self.capacity:
            raise ValueError(f"{max(rows)} rows exceed the capacity {self.capacity}")
        want = [max(0, -(-r // R) - h) for r, h in zip(rows, self._held)]
        if sum(want) > len(self._free):
            raise ValueError(f"{sum(want)} pages wanted, {len(self._free)} free: evict, release or build a larger pool")
        for s, n in enumerate(want):
            for _ in range(n):
                self._pages[s, self._held[s]] = self._free.pop()
                self._held[s] += 1
        if any(want):
            self.table.copy_(self._pages)

    def append(self, block: int, k: Tensor, v: Tensor, rows: Optional[Sequence[int]] = None) -> None:  # noqa: ANN001
        """Rows t < rows[s] (default all) of k, v [sequences, H, T, d] behind each sequence's last row of `block`."""
        self._own("append")
        S, NB, H, cap, D = self.shape
        if k.shape != v.shape or k.dim() != 4 or k.shape[0] != S or k.shape[1] != H or k.shape[3] != D:
            raise ValueError(f"append expects k/v [{S}, {H}, T, {D}], got {tuple(k.shape)} / {tuple(v.shape)}")
        self._check_rows(block, k, v)
        T = k.shape[2]
        new = [T] * S if rows is None else [int(r) for r in rows]
        if len(new) != S or any(not 0 <= r <= T for r in new):
            raise ValueError(f"rows must be {S} counts from 0 to {T}, got {new}")
        ends = [a + n for a, n in zip(self._rows[block], new)]
        self.reserve(ends)
        count = None if rows is None else torch.tensor(new, dtype=torch.int32, device=self.table.device)
        paged_append(self.keys[block], self.values[block], self.table, self.lengths[block], k, v, count, **self._scales_of(block))
        self._grown(block, T if count is None else count, T)
        self._rows[block] = ends

    def append_packed(self, block: int, k: Tensor, v: Tensor, rows: Sequence[int]) -> None:
        """append of packed rows k, v [total, H, d]: rows[0] rows of the first sequence, then rows[1] of the second, and so
        on; none is padded."""
        self._own("append_packed")
        S, NB, H, cap, D = self.shape
        new = [int(r) for r in rows]
        if len(new) != S or min(new, default=0) < 0:
            raise ValueError(f"rows must be {S} counts of at least 0, got {new}")
        total = sum(new)
        if k.shape != v.shape or k.shape != (total, H, D):
            raise ValueError(f"append_packed expects k/v [{total}, {H}, {D}], got {tuple(k.shape)} / {tuple(v.shape)}")
        self._check_rows(block, k, v)
        ends = [a + n for a, n in zip(self._rows[block], new)]
        self.reserve(ends)
        count = torch.tensor(new, dtype=torch.int32, device=self.table.device)
        slots, starts = paged_slots(self.table, self.lengths[block], count, total, self.keys.shape[1], self.page_rows)
        paged_append_packed(self.keys[block], self.values[block], self.table, self.lengths[block], count, k, v, slots, starts,
                            **self._scales_of(block))
        self._grown(block, count, max(new, default=0))
        self._rows[block] = ends

    def _check_rows(self, block: int, k: Tensor, v: Tensor) -> None:
        if k.dtype != self._row_dtype(k.dtype) or v.dtype != k.dtype:
            raise ValueError(f"append expects {self._row_dtype(k.dtype)} (cast before appending)")
        if not 0 <= block < self.shape[1]:
            raise ValueError(f"block {block} out of range [0, {self.shape[1]})")
        _no_grad("PagedIclKVCache.append", k, v)
        _nat.require_device(k, v, self.keys)

    def _scales_of(self, block: int) -> dict:
        return {} if self.scales is None else {"scales": self.scales[block]}

    def _grown(self, block: int, count, most: int) -> None:  # noqa: ANN001
        """The lengths (and bounds) of a block after an append of `count` rows per sequence, at most `most`."""
        lengths = self.lengths[block]
        if self.bounds is not None:
            paged_bounds(self.keys[block], self.table, lengths + count, self.bounds[block], self.bound_scales[block], lengths, most,
                         **self._scales_of(block))
        lengths += count

    def _row_dtype(self, dtype: torch.dtype) -> torch.dtype:
        if self.scales is None:
            return self.keys.dtype
        return dtype if dtype in (torch.bfloat16, torch.float32) else torch.bfloat16

    def _attn_dtype(self, dtype: torch.dtype) -> torch.dtype:
        return super()._attn_dtype(dtype) if self.scales is None else torch.promote_types(dtype, torch.bfloat16)

    def append_projected(self, block: int, x: Tensor, in_proj_weight: Tensor, in_proj_bias: Optional[Tensor] = None,
                         rows: Optional[Sequence[int]] = None) -> None:
        """append of the rows x [sequences, T, width] through the K|V thirds of a block's packed in-projection (one
        GEMM; the append reads the heads out of it through strides)."""
        self.append(block, *self._project_kv(x, in_proj_weight, in_proj_bias), rows)

    def query(self, block: int, q: Tensor, valid_kv_len: Optional[Union[int, Tensor]] = None,
              out: Optional[Tensor] = None) -> Tensor:
        """Attention of q [sequences, H, Tq, d] over `block` of the cache: each sequence's own rows, of those the ones
        below valid_kv_len if given (a number, or a tensor of one for all or one per sequence). q in the cache's dtype or one
        that widens to it, its heads as many as the cache's or a multiple (head h reads head h // (Hq // H) of the cache). No
        gradient, however many query rows there are. The bf16 probabilities take part as two bf16 terms in the pages, and as
        one where an untracked cache answers 256 rows and more (1,024 over all sequences, by many cached ones) with the dense
        kernel, as IclKVCache does: up to 2^-8 of each value then."""
        _no_grad("PagedIclKVCache.query", q, out)
        S, (_, _, H, _, D) = self.table.shape[0], self.keys.shape
        if q.dim() != 4 or q.shape[0] != S or q.shape[1] == 0 or q.shape[1] % H or q.shape[3] != D:
            raise ValueError(f"query expects q [{S}, {H} heads or a multiple, Tq, {D}], got {tuple(q.shape)}")
        lengths = self.default_valid(block)
        longest = max(self._lengths_of(block))
        captured = self._capturing()  # a replay meets the lengths of its time
        if isinstance(valid_kv_len, Tensor):
            valid = valid_kv_len.to(lengths.device).reshape(-1).expand_as(lengths)
            if valid.dtype is not torch.int32:  # compared in 64 bits: a cast first would wrap a number beyond 32 round
                valid = valid.to(torch.int64).clamp(min=0)
            lengths = torch.minimum(valid, lengths, out=torch.empty_like(lengths))
        elif valid_kv_len is not None and (captured or int(valid_kv_len) < longest):
            longest = max(0, min(int(valid_kv_len), self.capacity))
            lengths = lengths.clamp(max=longest)
        dt = self.keys.dtype if self.scales is None else self._attn_dtype(q.dtype)
        if torch.promote_types(q.dtype, dt) != dt or dt not in (torch.bfloat16, torch.float32):
            raise ValueError(f"q is {q.dtype}, wider than the {dt} cache: cast it")
        w = max(1, -(-longest // self.page_rows))
        if captured:
            w = self.table.shape[1]
        if self.select is not None and w > self.select:
            q, table, n = q.to(dt), self.table[:, :w], q.numel()
            if n > 32 * _SELECT_ROWS or n > 32 * _SPARSE_ROWS or n * (self.select + w) > 8 * _SELECT_BYTES:  # n: 32 a query row at least
                return self._selected_in_slices(block, q, table, lengths, out)
            return self._selected(block, q, table, lengths, out)
        if not captured and q.shape[2] >= _DENSE_QUERY_ROWS and S * q.shape[2] >= _DENSE_ALL_ROWS \
                and S * q.shape[2] * longest >= _DENSE_SCORES and D == 64 and q.shape[1] == H and dt == torch.bfloat16 \
                and self.weights is None:
            return self._gathered(block, q.to(dt), lengths, longest, out)
        weights = None if self.weights is None else self.weights[:, :w * self.page_rows]
        return paged_attention(q.to(dt), self.keys[block], self.values[block], self.table[:, :w], lengths, weights, None, out,
                               **self._scales_of(block))

    def _selected(self, block: int, q: Tensor, table: Tensor, lengths: Tensor, out: Optional[Tensor]) -> Tensor:
        """query over selected pages."""
        eight = self._scales_of(block)
        index = paged_select(q, self.bounds[block], self.bound_scales[block], table, lengths, self.page_rows, self.select)
        return paged_sparse_attention(q, self.keys[block], self.values[block], table, lengths, index, None, out, **eight)

    def _selected_in_slices(self, block: int, q: Tensor, table: Tensor, lengths: Tensor, out: Optional[Tensor]) -> Tensor:
        """_selected, as much at a time as the operators take and _SELECT_BYTES hold: runs of sequences, of one sequence runs of
        query rows."""
        (S, Hq, T, _), H = q.shape, self.keys.shape[2]
        each = 4 * H * self.select + max(0, int(_nat.load().tabicl_paged_select_workspace_bytes(1, H, 1, table.shape[1])))
        pairs = max(1, min(_SELECT_ROWS // H, _SPARSE_ROWS // Hq, _SELECT_BYTES // each))  # (sequence, query row) pairs of a slice
        ns = min(S, max(1, pairs // T))
        nt = pairs // ns
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        q = _apart(q, out)
        for s in range(0, S, ns):
            for t in range(0, T, nt):
                self._selected(block, q[s:s + ns, :, t:t + nt], table[s:s + ns], lengths[s:s + ns], out[s:s + ns, :, t:t + nt])
        return out

    def _gathered(self, block: int, q: Tensor, lengths: Tensor, longest: int, out: Optional[Tensor]) -> Tensor:
        """query by the dense kernel, over the rows of one run of sequences after the other side by side."""
        each = [min(n, longest) for n in self._lengths_of(block)]
        most = _GATHER_BYTES // (2 * q.shape[1] * q.shape[3] * q.element_size())  # cached rows of a run
        if out is not None:
            q = _apart(q, out)
        elif len(each) * longest > most:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        start, o = 0, None
        while start < len(each):
            stop, rows = start + 1, each[start]
            while stop < len(each) and (stop + 1 - start) * max(rows, each[stop]) <= most:
                rows = max(rows, each[stop])
                stop += 1
            rows = max(1, rows)
            run = slice(start, stop)
            k, v = paged_gather(self.keys[block], self.values[block], self.table[run, :-(-rows // self.page_rows)], lengths[run],
                                rows, **self._scales_of(block))
            o = self._dense(q[run], k, v, lengths[run], None if out is None else out[run])
            del k, v  # before the next run's
            start = stop
        return o if out is None else out

    def query_blocks(self, x: Tensor, blocks, valid_kv_len: Optional[Union[int, Tensor]] = None,  # noqa: ANN001
                     q_transform: Optional[Callable[[Tensor], Tensor]] = None,
                     activation: Callable[[Tensor], Tensor] = F.gelu) -> Tensor:
        """IclKVCache.query_blocks over the pages. No gradient: the layers around the attention would pass on their own part
        of it alone, so one of x or of any weight is refused here."""
        if torch.is_grad_enabled() or _fwd_level() >= 0:
            _no_grad("PagedIclKVCache.query_blocks", x, *(t for w in blocks for t in vars(w).values() if isinstance(t, Tensor)))
        return super().query_blocks(x, blocks, valid_kv_len, q_transform, activation)

    def evict(self, keep: Union[int, Sequence[int]], recent: int = 0) -> Tensor:
        """Cuts each sequence to at most keep rows (a number, or one per sequence), in every block alike: its `recent`
        last rows and the heaviest of the others (paged_evict by the tracked weights, which follow their rows). Last are the
        rows of the highest numbers: rows that an eviction moved into freed places are among the earlier ones from then on.
        Pages behind the kept rows, reserved ones too, go back to the pool. Returns index [sequences, K] int32: slot j now
        holds the old row index[s, j]."""
        self._own("evict")
        if self.weights is None:
            raise ValueError("evict needs a cache built with track=True")
        S = self.table.shape[0]
        if any(r != self._rows[0] for r in self._rows):
            raise ValueError("the blocks hold different rows: append to every block before evicting")
        keeps = [int(keep)] * S if isinstance(keep, int) else [int(n) for n in keep]
        if len(keeps) != S or min(keeps, default=0) < 0:
            raise ValueError(f"keep must be one count of at least 0, or {S} of them")
        have = self._rows[0]
        w = max(1, -(-max(have, default=0) // self.page_rows))
        kept = [min(h, n) for h, n in zip(have, keeps)]
        keep_n = None if isinstance(keep, int) else torch.tensor(kept, dtype=torch.int32, device=self.table.device)
        index, weights, lengths = paged_evict(self.keys, self.values, self.table[:, :w], self.lengths[0], self.weights,
                                              max(kept, default=0) if keep_n is None else keep_n, recent)
        index = index[:, :max(kept, default=0)]
        self.weights[:, :weights.shape[1]] = weights
        self.lengths.copy_(lengths.expand_as(self.lengths))
        self._rows = [list(kept) for _ in self._rows]
        self._give_back(kept)
        return index

    def release(self, sequence: int) -> None:
        """Forgets a sequence: its pages go back to the pool, its place can be filled anew."""
        self._own("release")
        sequence = range(len(self._held))[sequence]
        for rows in self._rows:
            rows[sequence] = 0
        self.lengths[:, sequence] = 0
        if self.weights is not None:
            self.weights[sequence] = 0.0
        self._give_back([0 if s == sequence else held * self.page_rows for s, held in enumerate(self._held)])

    def _give_back(self, rows) -> None:  # noqa: ANN001
        """Pages past each sequence's first `rows` rows back to the pool."""
        changed = False
        for s, r in enumerate(rows):
            need = -(-r // self.page_rows)
            for p in range(self._held[s] - 1, need - 1, -1):
                self._free.append(int(self._pages[s, p]))
                self._pages[s, p] = -1
                changed = True
            self._held[s] = min(self._held[s], need)
        if changed:
            self.table.copy_(self._pages)

    def estimators(self, start: int, stop: int) -> "PagedIclKVCache":
        """Sequences [start, stop) as a cache of their own that answers queries (query_chunked): views of the pool, the
        table, the lengths and the tracked weights."""
        S = self.table.shape[0]
        if not 0 <= start < stop <= S:
            raise ValueError(f"estimators [{start}, {stop}) out of range [0, {S})")
        view = object.__new__(PagedIclKVCache)
        view.__dict__.update(self.__dict__)
        view.table = self.table[start:stop]
        view.lengths = self.lengths[:, start:stop]
        view.weights = None if self.weights is None else self.weights[start:stop]
        view._first = self._first + start
        return view

    def block_kv(self, block: int):
        """The block's pools [pages, H, page_rows, d]."""
        return self.keys[block], self.values[block]
