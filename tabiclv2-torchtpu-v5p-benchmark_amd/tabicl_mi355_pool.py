"""Checks that the operators of the paged K/V cache share (tabicl_mi355_paged, _paged8, _sparse, _books): a pool with its page
table and lengths, rows of K, V and queries, gradients that a serving operator has not got."""
from __future__ import annotations

from typing import Optional

import torch
import torch.autograd.forward_ad as _fwd
from torch import Tensor

import tabicl_mi355_native as _nat

# dtypes of 8-bit pools, with the library's codes
CODES = {torch.float8_e4m3fn: 0, torch.int8: 1}


# A call of few rows is over in 10 us on the GPU; the checks below take 4 us of a host core (12 with a test and a generator
# expression per property).
def rows16(t: Tensor, es: int):
    """(t, its (n, h, row) element strides) of [N, H, T, D] when its last dim is contiguous and it starts, and its other
    dims step, in multiples of 16 bytes (what the kernels' loads need), else of a contiguous copy. A dim of one entry,
    whose stride says nothing, counts as stride 0."""
    n, h, r, d = t.stride()
    shape = t.shape
    n, h, r = n if shape[0] > 1 else 0, h if shape[1] > 1 else 0, r if shape[2] > 1 else 0
    if (d == 1 or shape[3] == 1) and ((n | h | r) * es | t.data_ptr()) & 15 == 0:
        return t, n, h, r
    t = t.clone(memory_format=torch.contiguous_format)
    return t, shape[1] * shape[2] * shape[3], shape[2] * shape[3], shape[3]


def table_args(table: Tensor, lengths: Tensor) -> tuple:
    """Checks a page table with its lengths; returns (table, table stride, max_pages) as the entry points take them, and N."""
    ts = table.shape
    if table.dtype is not torch.int32 or len(ts) != 2 or (table.stride(1) != 1 and ts[1] > 1):
        raise ValueError("table must be an int32 [N, max_pages] tensor with contiguous rows")
    N, M = ts
    counts(lengths, N, "lengths")
    return (table.data_ptr(), table.stride(0) if N > 1 else M, M), N


def counts(t: Tensor, N: int, what: str) -> None:
    if t.dtype is not torch.int32 or t.shape != (N,) or (N > 1 and t.stride(0) != 1):
        raise ValueError(f"{what} must be a contiguous int32 tensor of {N} entries")


def pool_args(k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, lead: int = 0):
    """Checks a pool [pages, H, page_rows, D] (behind `lead` more dims) with its table and lengths; returns (pages, page
    stride, page_rows, table, table stride, max_pages) as the entry points take them, then H, D, N, device index."""
    shape, st = k_pages.shape, k_pages.stride()
    if len(shape) != 4 + lead or v_pages.shape != shape or v_pages.stride() != st:
        raise ValueError(f"k_pages and v_pages must be [{'blocks, ' * lead}pages, H, page_rows, D] of one layout, got "
                         f"{tuple(shape)} and {tuple(v_pages.shape)}")
    P, H, R, D = shape[lead:]
    if st[-1] != 1 or st[-2] != D or (st[-3] != R * D and H > 1):
        raise ValueError("a page [H, page_rows, D] must be contiguous")
    if k_pages.dtype is not v_pages.dtype:
        raise ValueError("k_pages and v_pages must share a dtype")
    ts = table.shape  # table_args' checks in place: a call of it takes as long as half of the checks here
    if table.dtype is not torch.int32 or len(ts) != 2 or (table.stride(1) != 1 and ts[1] > 1):
        raise ValueError("table must be an int32 [N, max_pages] tensor with contiguous rows")
    N, M = ts
    if lengths.dtype is not torch.int32 or lengths.shape != (N,) or (N > 1 and lengths.stride(0) != 1):
        raise ValueError(f"lengths must be a contiguous int32 tensor of {N} entries")
    dev = k_pages.get_device()
    if v_pages.get_device() != dev or table.get_device() != dev or lengths.get_device() != dev:
        raise ValueError("the pool, table and lengths must be on one device")
    return (P, st[lead] if P > 1 else H * R * D, R, table.data_ptr(), table.stride(0) if N > 1 else M, M), H, D, N, dev


def dense_code(dtype: torch.dtype) -> int:
    """The library's code of a bf16 or fp32 pool."""
    if dtype is torch.bfloat16:
        return _nat.DTYPE_BF16
    if dtype in CODES:
        raise ValueError("a pool of 8-bit codes needs its scales [pages, H, 2]")
    return _nat.dtype_code(dtype)


def check_scales(scales: Optional[Tensor], P: int, H: int, dev: int) -> None:
    if scales is None:
        raise ValueError("a pool of 8-bit codes needs its scales [pages, H, 2]")
    if scales.dtype is not torch.float32 or scales.shape != (P, H, 2) or not scales.is_contiguous() or scales.data_ptr() & 7 \
            or scales.get_device() != dev:
        raise ValueError(f"scales must be a contiguous float32 [{P}, {H}, 2] tensor on the pool's device, got {scales.dtype} "
                         f"{tuple(scales.shape)}")


def pool_format(k_pages: Tensor, scales: Optional[Tensor], dev: int) -> int:
    """The library's pool format (0 bf16, 1 fp32, 2 e4m3, 3 int8); scales belong to the 8-bit ones alone."""
    code = CODES.get(k_pages.dtype)
    if code is None:
        if scales is not None:
            raise ValueError(f"scales are for pools of 8-bit codes, not {k_pages.dtype}")
        return _nat.dtype_code(k_pages.dtype)
    check_scales(scales, k_pages.shape[0], k_pages.shape[1], dev)
    return 2 + code


def query_args(q: Tensor, out: Tensor, N: int, H: int, D: int, dev: int) -> tuple:
    """Checks queries and their output; returns out's (n, h, row) strides."""
    shape = q.shape
    if len(shape) != 4 or shape[0] != N or shape[3] != D or shape[1] % max(1, H):
        raise ValueError(f"q must be [{N}, a multiple of {H} heads, Tq, {D}], got {tuple(shape)}")
    if out.shape != shape or out.dtype is not q.dtype:
        raise ValueError("out must match q")
    if q.get_device() != dev or out.get_device() != dev:
        raise ValueError("q, out and the pool must be on one device")
    on, oh, orow, od = out.stride()
    Hq, Tq = shape[1], shape[2]
    if od != 1 or (N > 1 and on == 0) or (Hq > 1 and oh == 0) or (Tq > 1 and orow == 0):
        raise ValueError("out needs a contiguous last dim and a place of its own for each row")
    return on if N > 1 else 0, oh if Hq > 1 else 0, orow if Tq > 1 else 0


def apart(q: Tensor, out: Tensor) -> Tensor:
    """q, or a copy of it where `out` may overlap it: the kernels read q again after parts of the output are written (the
    weights, and the tiles of one item in several workgroups)."""
    return q.clone() if q.untyped_storage().data_ptr() == out.untyped_storage().data_ptr() else q


def elsewhere(dev: int, *ts: Tensor) -> bool:
    """Whether tensors of device `dev` are not on the current one, by which a HIP launch goes; raises for the CPU."""
    if dev >= 0 and dev == torch.cuda.current_device():
        return False
    _nat.require_device(*ts)
    return True


def workspace(nbytes: int, what: str, like: Tensor) -> tuple:
    """(a tensor to hold on to, its address, its bytes); raises what the size function refused."""
    if nbytes < 0:
        raise _nat.UnsupportedShapeError(f"{what}: {_nat.last_error()}")
    if nbytes == 0:
        return None, None, 0
    ws = torch.empty(nbytes, dtype=torch.uint8, device=like.device)
    return ws, ws.data_ptr(), nbytes


def fwd_level() -> int:
    return getattr(_fwd, "_current_level", 0)


def no_grad(what: str, *ts: Optional[Tensor]) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts):
        raise ValueError(f"{what} has no gradient (a serving operator): detach its inputs or call it under no_grad")
    # forward mode: an op without a formula would drop the tangent and say nothing
    if fwd_level() >= 0 and any(t is not None and _fwd.unpack_dual(t).tangent is not None for t in ts):
        raise ValueError(f"{what} has no gradient, nor one in forward mode (a serving operator): detach its inputs")
