"""The 8-bit paged K/V cache, attention over selected pages and the books of a pool on the GPU as timed cases: attention
over pages of e4m3 or int8 values with a scale for each page and head, rows written into and read back from such pages,
the bounds of the keys of each page, the selection of the pages that each query row attends to with the attention over
them, and page tables and slot maps from request lengths.

listed() names the cases; draw(rng) gives another one of the same ranges; prepare / run / work take a case. Where
`own` is false, run() computes an operator from elementary torch operations in fp32 (whole numbers: exactly); where it is
true, it calls the package. exact() restates a case in float64 and in Python integers. Inputs come from torch's device
generator and the seed alone.

Scales are powers of two: 2^k is the smallest with max |x| <= Q 2^k (Q: 448 for e4m3, 127 for int8 and for bounds), k in
[-60, 100]. A page that is added to keeps the larger of its scale and that of the new rows; the rows that it holds are
rounded again where the scale grows.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tabiclv2-torchtpu-v5p-benchmark_amd")
DT = {"bf16": torch.bfloat16, "fp32": torch.float32, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}
ES = {"bf16": 2, "fp32": 4, "e4m3": 1, "int8": 1}
TOP = {"e4m3": 448, "int8": 127}
HEADS, DIM = 8, 64  # the ICL stage


def _paged():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import tabicl_mi355_paged
    return tabicl_mi355_paged


# ---------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------
def _cache(name, kind, seqs, shortest, longest, rows=1, pool="bf16", dtype="bf16", kv_heads=HEADS, group=1, dim=DIM, page=64,
           select=0):
    return {"name": name, "kind": kind, "seqs": seqs, "shortest": shortest, "longest": longest, "rows": rows, "pool": pool,
            "dtype": dtype, "kv_heads": kv_heads, "group": group, "dim": dim, "page": page, "select": select}


def _fill(name, seqs, start, rows, pool, dtype="bf16", kv_heads=HEADS, dim=DIM, page=64):
    return {"name": name, "kind": "fill", "seqs": seqs, "start": start, "rows": rows, "pool": pool, "dtype": dtype,
            "kv_heads": kv_heads, "dim": dim, "page": page}


def _books(name, seqs, held, new, page=64):
    return {"name": name, "kind": "books", "seqs": seqs, "held": held, "new": new, "page": page}


def listed() -> list:
    return [
        # one test row of a small table, 8 estimators, as a service answers it (latency)
        _cache("q8_one_small", "attn", 8, 700, 700, pool="e4m3"),
        # one test row at the headline table: 45,000 cached train rows in 8 bits
        _cache("q8_one_large", "attn", 8, 45000, 45000, pool="int8"),
        # a mixed batch in validation precision: odd lengths, grouped heads of 128 dims, small pages
        _cache("q8_ragged_fp32", "attn", 16, 501, 10001, rows=3, pool="e4m3", dtype="fp32", group=4, dim=128, page=32),
        # one new row per sequence into a page that is partly full, and the cache read back as the dense kernels take it
        _fill("fill_one", 8, 1000, 1, "e4m3"),
        # a block's train rows at fit time, and read back for a large batch of test rows
        _fill("fill_fit", 8, 0, 45000, "int8"),
        # the keys' bounds of a small cache's pages; of the headline one
        _cache("bounds_small", "bounds", 8, 1000, 1000),
        _cache("bounds_large", "bounds", 8, 45000, 45000),
        # one test row at the headline table that reads a tenth of it
        _cache("sparse_one", "sparse", 8, 45000, 45000, select=64),
        # a few test rows over an 8-bit cache
        _cache("sparse_q8", "sparse", 8, 20001, 20001, rows=4, pool="e4m3", select=32),
        # a mixed batch with grouped heads, some of its tables smaller than the selection
        _cache("sparse_ragged", "sparse", 32, 300, 30000, kv_heads=4, group=4, dim=128, page=32, select=48),
        # a serving step: one new row for each of 256 requests
        _books("books_step", 256, 8000, 1),
        # 64 requests that arrive with up to 10,000 rows each
        _books("books_fit", 64, 0, 10000),
    ]


def _log(rng, lo: int, hi: int) -> int:
    """An integer spread evenly over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    kind = rng.choice(["attn", "attn", "fill", "bounds", "sparse", "sparse", "books"])
    page = rng.choice([16, 32, 64, 128, 256])
    seqs = _log(rng, 1, 64)
    if kind == "books":
        seqs = _log(rng, 1, 2000)
        held = rng.choice([0, _log(rng, 1, 10000)])
        return {"kind": kind, "seqs": seqs, "held": held, "new": _log(rng, 1, max(1, min(10000, 640000 // seqs))), "page": page}
    kv_heads, dim = rng.choice([(8, 64), (8, 64), (4, 32), (8, 32), (8, 128), (2, 128)])
    pool = rng.choice(["e4m3", "int8"] if kind in ("attn", "fill") else ["bf16", "bf16", "fp32", "e4m3", "int8"])
    dtype = pool if pool in ("bf16", "fp32") else rng.choice(["bf16", "bf16", "fp32"])
    case = {"kind": kind, "seqs": seqs, "pool": pool, "dtype": dtype, "kv_heads": kv_heads, "dim": dim, "page": page}
    values = seqs * kv_heads * dim * 2  # of one cached row of every sequence, K and V
    if kind == "fill":
        rows = _log(rng, 1, max(1, min(50000, 180000000 // values // (1 if dtype == "bf16" else 2))))
        return {**case, "start": rng.choice([0, rng.randint(1, 2000)]), "rows": rows}
    longest = _log(rng, 1, max(1, min(50000, 360000000 // values // ES[pool])))
    case = {**case, "shortest": max(1, int(longest * rng.choice([1.0, rng.random()]))), "longest": longest, "rows": 1, "group": 1,
            "select": 0}
    if kind == "bounds":
        return case
    group = rng.choice([1, 1, 2, 4])
    if kind == "attn":
        most = 46000000 // (seqs * kv_heads * group * longest)
        return {**case, "group": group, "rows": _log(rng, 1, max(1, min(64, most)))}
    select = rng.randint(1, max(1, min(64, -(-longest // page), 16384 // page)))
    most = 30000000 // (seqs * kv_heads * select * page)  # rows of selected pages over all query rows
    return {**case, "group": group, "select": select, "rows": _log(rng, 1, max(1, min(32, most)))}


def _lengths(case) -> list:
    """The sequences' lengths, spread evenly over the logarithm from the shortest to the longest."""
    lo, hi, n = case["shortest"], case["longest"], case["seqs"]
    return [round(lo * (hi / lo) ** (i / (n - 1))) if n > 1 else hi for i in range(n)]


def _news(case) -> list:
    """The rows that the requests get: from half of `new` to all of it."""
    n, new = case["seqs"], case["new"]
    return [(new + 1) // 2 + (new // 2) * i // max(1, n - 1) for i in range(n)]


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def prepare(case, seed: int) -> dict:
    """Pages in random order behind a page table, as a cache that has been in use for a while holds them. Heads differ in
    size and sharpness, and in some the dims do, as keys after a learned projection do."""
    dev = torch.device("cuda", 0)
    g = torch.Generator(device=dev).manual_seed(1000003 * (seed + 1))
    if case["kind"] == "books":
        return _prepare_books(case, g, dev)
    R, H, D, N, pool = case["page"], case["kv_heads"], case["dim"], case["seqs"], case["pool"]

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device=dev, dtype=dtype)

    if case["kind"] == "fill":
        held, total = [case["start"]] * N, [case["start"] + case["rows"]] * N
    else:
        order = torch.randperm(N, generator=g, device=dev).tolist()
        held = total = [_lengths(case)[i] for i in order]
    width = -(-max(total) // R)
    P = N * width + 3
    ids = torch.randperm(P, generator=g, device=dev)[: N * width].to(torch.int32)
    s = {"case": case, "table": ids.view(N, width), "lengths": torch.tensor(held, dtype=torch.int32, device=dev)}
    size = torch.exp(randn(H, 1, D) * 0.5)  # per head and dim
    if pool in TOP:
        # codes over the whole range of their type as pages of normal values have them, a scale per page and head
        s["scales"] = torch.exp2(torch.randint(-9, -4, (P, H, 2), generator=g, device=dev).float())
        s["k_pages"], s["v_pages"] = (_to_pool(randn(P, H, R, D, dtype=torch.bfloat16).float() * TOP[pool] / 4.5, pool)
                                      for _ in range(2))
    else:
        s["scales"] = None
        s["k_pages"] = (randn(P, H, R, D, dtype=DT[pool]) + randn(P, H, 1, D, dtype=DT[pool])).mul_(size.to(DT[pool]))
        s["v_pages"] = randn(P, H, R, D, dtype=DT[pool]) if case["kind"] == "sparse" else None
    if case["kind"] == "fill":
        # heads read out of a K|V projection [N, T, 2, H, D]
        kv = randn(N, case["rows"], 2, H, D, dtype=DT[case["dtype"]])
        s["k"], s["v"] = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
        return s
    if case["kind"] == "bounds":
        s["v_pages"] = None
        s["bounds"] = torch.zeros(P, H, 2, D, dtype=torch.int8, device=dev)
        s["bound_scales"] = torch.zeros(P, H, device=dev)
        return s
    q = randn(N, H * case["group"], case["rows"], D) * torch.exp(randn(N, H * case["group"], 1, 1) * 0.5)
    s["q"] = q.to(DT[case["dtype"]])
    if case["kind"] == "sparse":
        s["bounds"], s["bound_scales"] = _bounds_of(_pool_values(s["k_pages"], s["scales"], 0), _live(s))
    return s


def _prepare_books(case, g, dev) -> dict:
    """Requests that hold up to `held` rows and get up to `new` ones; the pool's free pages in any order on their stack. The
    slot map has a few places more than there are rows, as one of a fixed size (a captured graph's) has."""
    N, R = case["seqs"], case["page"]
    order = torch.randperm(N, generator=g, device=dev).cpu()
    lengths = torch.randint(case["held"] // 2, case["held"] + 1, (N,), generator=g, device=dev)
    count = torch.tensor(_news(case))[order].to(dev)
    width = -(-(case["held"] + case["new"]) // R)
    has = (lengths + R - 1) // R
    P = N * width + 17
    ids = torch.randperm(P, generator=g, device=dev).to(torch.int32)
    table = torch.full((N, width), -1, dtype=torch.int32, device=dev)
    mine = torch.arange(width, device=dev) < has[:, None]
    used = int(has.sum())
    table[mine] = ids[:used]
    free = torch.zeros(P, dtype=torch.int32, device=dev)
    free[: P - used] = ids[used:]
    return {"case": case, "table": table, "lengths": lengths.to(torch.int32), "count": count.to(torch.int32), "free": free,
            "free_count": torch.tensor([P - used], dtype=torch.int32, device=dev), "total": sum(_news(case)) + 5}


# ---------------------------------------------------------------------------------------------
# 8-bit values and bounds, in elementary operations
# ---------------------------------------------------------------------------------------------
def _pow2_scale(most, top):
    """The smallest 2^k with most <= top 2^k, k in [-60, 100]."""
    mant, exp = torch.frexp(most)  # most = mant 2^exp, mant in [1/2, 1)
    limit, shift = torch.frexp(torch.tensor(float(top)))
    k = (exp - int(shift) + (mant > float(limit)).to(exp.dtype)).clamp(-60, 100)
    return torch.ldexp(torch.ones_like(most), torch.where(most > 0, k, -60))


def _to_pool(x, pool):
    """x rounded to the pool's values, saturating."""
    if pool == "int8":
        return torch.nan_to_num(x, nan=0.0, posinf=127.0, neginf=-127.0).clamp_(-127, 127).round_().to(torch.int8)
    return x.clamp(-448, 448).to(torch.float8_e4m3fn)


def _pool_values(pages, scales, which):
    """The values of the pages in fp32; which: 0 K, 1 V."""
    return pages.float() if scales is None else pages.float() * scales[:, :, which, None, None]


def _take(pages, ids):
    """pages[ids], for 8-bit floats too."""
    return pages.view(torch.uint8)[ids].view(pages.dtype) if pages.dtype is torch.float8_e4m3fn else pages[ids]


def _live(s):
    """[pages, page rows]: whether a sequence has a row there."""
    kp, table, lengths = s["k_pages"], s["table"], s["lengths"]
    P, R = kp.shape[0], kp.shape[2]
    live = torch.zeros(P, R, dtype=torch.bool, device=kp.device)
    at = torch.arange(table.shape[1] * R, device=kp.device).view(1, -1, R)
    live[table.long()] = at < lengths[:, None, None]
    return live


def _bounds_of(k, live):
    """The bounds [pages, H, 2, D] (the largest of each dim rounded up, the smallest rounded down, in int8 steps of the
    page's and head's scale) of keys k [pages, H, R, D] at the live rows, and the scales [pages, H]."""
    at = live[:, None, :, None]
    hi = torch.where(at, k, -math.inf).amax(2)
    lo = torch.where(at, k, math.inf).amin(2)
    empty = ~live.any(1)[:, None, None]
    hi, lo = hi.masked_fill(empty, 0.0), lo.masked_fill(empty, 0.0)
    scale = _pow2_scale(torch.maximum(hi.abs(), lo.abs()).amax(2), 127)
    both = torch.stack((torch.ceil(hi / scale[..., None]), torch.floor(lo / scale[..., None])), dim=2)
    return both.to(torch.int8), scale


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(s):
    return {"attn": _run_attn, "fill": _run_fill, "bounds": _run_bounds, "sparse": _run_sparse, "books": _run_books}[
        s["case"]["kind"]](s)


def _run_attn(s):
    q, kp, vp, table, lengths, scales = s["q"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], s["scales"]
    if own:
        return {"out": _paged().paged_attention(q, kp, vp, table, lengths, scales=scales)}
    N, Hq, T, D = q.shape
    H, R = kp.shape[1], kp.shape[2]
    L = table.shape[1] * R
    rows = table.long()

    def side(pages, which):
        x = _take(pages, rows).float() * scales[rows][..., which, None, None]
        return x.permute(0, 2, 1, 3, 4).reshape(N, H, L, D)

    live = (torch.arange(L, device=q.device) < lengths[:, None]).view(N, 1, 1, L)
    scores = torch.matmul(q.float().reshape(N, H, -1, D), side(kp, 0).transpose(2, 3)) * D ** -0.5
    scores = torch.where(live, scores, -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    return {"out": torch.matmul(p, side(vp, 1)).view(N, Hq, T, D).to(q.dtype)}


def _run_fill(s):
    kp, vp, table, lengths, scales = s["k_pages"], s["v_pages"], s["table"], s["lengths"], s["scales"]
    k, v, c = s["k"], s["v"], s["case"]
    rows = c["start"] + c["rows"]
    if own:
        _paged().paged_append(kp, vp, table, lengths, k, v, scales=scales)
        k_rows, v_rows = _paged().paged_gather(kp, vp, table, lengths + c["rows"], rows, scales=scales, dtype=k.dtype)
        return {"k": k_rows, "v": v_rows, "scales": scales}
    N, H, T, D = k.shape
    R, pool = kp.shape[2], c["pool"]
    first, kept = c["start"] // R, c["start"] % R  # the first page that is written, and the rows it holds already
    width = table.shape[1] - first
    ids = table[:, first:].long()
    new = torch.arange(width * R, device=k.device)
    new = ((new >= kept) & (new < kept + T)).view(1, width, 1, R, 1)
    for which, pages, x in ((0, kp, k), (1, vp, v)):
        held = _take(pages, ids).float() * scales[ids][..., which, None, None]  # [N, width, H, R, D]
        x = torch.nn.functional.pad(x.float(), (0, 0, kept, width * R - kept - T)).view(N, H, width, R, D).transpose(1, 2)
        scale = _pow2_scale(torch.where(new, x.abs(), 0.0).amax((3, 4)), TOP[pool])
        if kept:
            scale[:, 0] = torch.maximum(scale[:, 0], scales[ids[:, 0]][..., which])
        codes = _to_pool(torch.where(new, x, held) / scale[..., None, None], pool)
        pages.view(torch.uint8)[ids] = codes.view(torch.uint8)
        scales[..., which][ids] = scale
    full = table.long()
    k_rows, v_rows = ((_take(p, full).float() * scales[full][..., which, None, None]).transpose(1, 2)
                      .reshape(N, H, -1, D)[:, :, :rows].to(k.dtype) for which, p in ((0, kp), (1, vp)))
    return {"k": k_rows, "v": v_rows, "scales": scales}


def _run_bounds(s):
    if own:
        _paged().paged_bounds(s["k_pages"], s["table"], s["lengths"], s["bounds"], s["bound_scales"], scales=s["scales"])
    else:
        both, scale = _bounds_of(_pool_values(s["k_pages"], s["scales"], 0), _live(s))
        pages = s["table"].long()
        pages = pages[torch.arange(pages.shape[1], device=pages.device) * s["case"]["page"] < s["lengths"][:, None]]
        s["bounds"][pages], s["bound_scales"][pages] = both[pages], scale[pages]
    return {"bounds": s["bounds"].float() * s["bound_scales"][..., None, None]}


def _run_sparse(s):
    q, kp, vp, table, lengths, scales, c = (s["q"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], s["scales"],
                                           s["case"])
    if own:
        index = _paged().paged_select(q, s["bounds"], s["bound_scales"], table, lengths, c["page"], c["select"])
        return {"index": index,
                "out": _paged().paged_sparse_attention(q, kp, vp, table, lengths, index, scales=scales)}
    N, Hq, T, D = q.shape
    H, R, M, K = kp.shape[1], kp.shape[2], table.shape[1], c["select"]
    G = Hq // H
    qg = q.float().view(N, H, G, T, D)
    # the bound of each page: products of whole numbers, exact in fp32
    step = _pow2_scale(qg.abs().amax((2, 4), keepdim=True), 127)
    whole = torch.round(qg / step).clamp(-127, 127)
    rows = table.long()
    both = s["bounds"][rows].float().permute(0, 2, 3, 4, 1)  # [N, H, 2, D, M]
    bound = torch.matmul(whole.clamp(min=0).view(N, H, G * T, D), both[:, :, 0]) \
        + torch.matmul(whole.clamp(max=0).view(N, H, G * T, D), both[:, :, 1])
    bound = bound.view(N, H, G, T, M).amax(2) * s["bound_scales"][rows].transpose(1, 2)[:, :, None]
    some = (torch.arange(M, device=q.device) * R < lengths[:, None]).view(N, 1, 1, M)
    order = torch.sort(torch.where(some, bound, -math.inf), dim=-1, descending=True, stable=True).indices[..., :K]
    order = torch.sort(torch.where(some.expand(bound.shape).gather(3, order), order, M), dim=-1).values
    index = torch.where(order < M, order, -1).int()
    if order.shape[3] < K:
        index = torch.nn.functional.pad(index, (0, K - order.shape[3]), value=-1)
    # the rows of the chosen pages, 0 for every other query row's
    at = order.clamp(max=M - 1)
    page = rows.view(N, 1, 1, M).expand(N, H, T, M).gather(3, at)  # [N, H, T, K]
    live = (at[..., None] * R + torch.arange(R, device=q.device) < lengths.view(N, 1, 1, 1, 1)) & (order < M)[..., None]
    heads = torch.arange(H, device=q.device).view(1, H, 1, 1)

    def side(pages, which):
        flat = pages.view(-1, R, D)
        x = _take(flat, page * H + heads).float()
        if scales is not None:
            x = x * scales[page, heads, which][..., None, None]
        return x.view(N, H, T, -1, D)

    scores = torch.matmul(qg.transpose(2, 3), side(kp, 0).transpose(3, 4)) * D ** -0.5  # [N, H, T, G, K R]
    scores = torch.where(live.view(N, H, T, 1, -1), scores, -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    out = torch.matmul(p, side(vp, 1)).transpose(2, 3).reshape(N, Hq, T, D)
    return {"index": index, "out": out.to(q.dtype)}


def _run_books(s):
    """Pages for the new rows, where each row goes, and (the request is done) the new pages back on the stack."""
    table, lengths, count, free, free_count, R = (s["table"], s["lengths"], s["count"], s["free"], s["free_count"],
                                                  s["case"]["page"])
    P, (N, M) = free.shape[0], table.shape
    if own:
        granted = _paged().paged_reserve(table, lengths, count, free, free_count, R)
        slots, starts = _paged().paged_slots(table, lengths, count, s["total"], P, R)
        given = table.clone()
        _paged().paged_release(table, lengths, free, free_count, R)
        return {"granted": granted, "slots": slots, "starts": starts, "given": given, "table": table, "free": free,
                "free_count": free_count}
    at = torch.arange(M, device=table.device)
    has, end = (lengths.long() + R - 1) // R, (lengths.long() + count + R - 1) // R
    none = (table < 0) | (table >= P)
    want = (at >= has[:, None]) & (at < end[:, None]) & none
    rank = want.view(-1).long().cumsum(0).view(N, M) - 1
    gets = want & (rank < free_count)
    top = (free_count.long() - 1 - rank).clamp(0, P - 1)
    given = torch.where(gets, free[top], table)
    left = free_count - gets.sum()
    missing = (at >= has[:, None]) & (at < end[:, None]) & ((given < 0) | (given >= P))
    first = torch.where(missing, at, M).amin(1)  # the first page that is not there
    granted = torch.minimum(first * R - lengths, count.long()).clamp(min=0).int()
    ends = count.long().cumsum(0)
    starts = torch.nn.functional.pad(ends, (1, 0)).int()
    j = torch.arange(s["total"], device=table.device)
    seq = torch.searchsorted(ends, j, right=True).clamp(max=N - 1)
    row = lengths.long()[seq] + j - starts.long()[seq]
    page = given.long()[seq, (row // R).clamp(max=M - 1)]
    slots = torch.where((page >= 0) & (page < P) & (j < ends[-1]), page * R + row % R, -1)
    # back: the last page given is the first one on the stack again
    out = (at >= has[:, None]) & (given >= 0) & (given < P)
    n = out.sum()
    back = out.view(-1).long().cumsum(0).view(N, M) - 1
    to = torch.where(out, left + n - 1 - back, P)
    stack = torch.cat((free, free[:1]))
    stack.scatter_(0, to.view(-1), given.view(-1))
    free.copy_(stack[:P])
    table.copy_(torch.where(out, -1, given))
    free_count.copy_(left + n)
    return {"granted": granted, "slots": slots, "starts": starts, "given": given, "table": table, "free": free,
            "free_count": free_count}


def work(case) -> dict:
    """Each input read once and each output written once; of a selection the bounds of every page, and K and V of the pages
    that are chosen (each once: as many as there are, where the query rows together choose more)."""
    if case["kind"] == "books":
        rows = sum(_news(case))
        pages = case["seqs"] + rows // case["page"]
        return {"bytes": 8 * rows + 16 * pages + 16 * case["seqs"], "flops": 0}
    H, D, R, N = case["kv_heads"], case["dim"], case["page"], case["seqs"]
    row = H * D * ES[case["pool"]] * 2  # of a cached row, K and V
    if case["kind"] == "fill":
        wide = H * D * ES[case["dtype"]] * 2
        return {"bytes": N * (case["rows"] * (wide + row) + (case["start"] + case["rows"]) * (row + wide)), "flops": 0}
    lengths = _lengths(case)
    pages = sum(-(-n // R) for n in lengths)
    if case["kind"] == "bounds":
        return {"bytes": sum(lengths) * row // 2 + pages * H * 2 * D, "flops": 0}
    heads = H * case["group"]
    ends = 2 * N * heads * case["rows"] * D * ES[case["dtype"]]
    if case["kind"] == "attn":
        return {"bytes": sum(lengths) * row + ends, "flops": 4 * sum(lengths) * heads * case["rows"] * D}
    each = [min(n, case["select"] * R) for n in lengths]
    once = sum(min(n, e * case["rows"]) for n, e in zip(lengths, each))
    return {"bytes": once * row + pages * H * 2 * D + ends + 4 * N * H * case["rows"] * case["select"],
            "flops": 4 * case["rows"] * heads * D * (sum(each) + pages)}


# ---------------------------------------------------------------------------------------------
# float64 and whole numbers
# ---------------------------------------------------------------------------------------------
def exact(case, seed: int):
    s = prepare(case, seed)
    return {"attn": _exact_attn, "fill": _exact_fill, "bounds": _exact_bounds, "sparse": _exact_sparse,
            "books": _exact_books}[case["kind"]](case, s)


def _rows64(s, which, n, at):
    """K (0) or V (1) of rows `at` of sequence n in float64: [rows, H, D]."""
    pages = s["v_pages"] if which else s["k_pages"]
    R = pages.shape[2]
    ids = s["table"][n].long()[at // R]
    x = pages.view(torch.uint8)[ids, :, at % R].view(pages.dtype) if pages.dtype is torch.float8_e4m3fn else pages[ids, :, at % R]
    return x.float().double() if s["scales"] is None else x.float().double() * s["scales"].double()[ids][:, :, which, None]


def _softmax_product(q, k, v, dim):
    return torch.softmax(q.double() @ k.t() / math.sqrt(dim), dim=-1) @ v


def _exact_attn(case, s):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for n, count in enumerate(s["lengths"].tolist()):
        at = torch.arange(count, device=out.device)
        k, v = _rows64(s, 0, n, at), _rows64(s, 1, n, at)
        for h in range(out.shape[1]):
            out[n, h] = _softmax_product(s["q"][n, h], k[:, h // case["group"]], v[:, h // case["group"]], case["dim"])
    return {"out": out}


def _scale64(most, top):
    """The smallest 2^k with most <= top 2^k, k in [-60, 100], by trying."""
    scale = torch.full_like(most, 2.0 ** -60)
    for _ in range(160):
        scale = torch.where(most > top * scale, scale * 2, scale)
    return scale


def _round64(x, pool):
    """x to the nearest value of the pool, ties to the even one."""
    if pool == "int8":
        return torch.round(x).clamp(-127, 127)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)  # 4 significant bits, 2^-9 at least
    return (torch.round(x / step) * step).clamp(-448, 448)


def _exact_fill(case, s):
    R, N, start, T, pool = case["page"], case["seqs"], case["start"], case["rows"], case["pool"]
    scales = s["scales"].double()
    rows = start + T
    out = []
    for which, x in ((0, s["k"]), (1, s["v"])):
        held = [None] * N
        for n in range(N):
            val = torch.zeros(rows, case["kv_heads"], case["dim"], dtype=torch.float64, device=x.device)
            if start:
                val[:start] = _rows64(s, which, n, torch.arange(start, device=x.device))
            val[start:] = x[n].transpose(0, 1).double()
            first = start - start % R
            pad = -(rows - first) % R
            part = torch.nn.functional.pad(val[first:], (0, 0, 0, 0, 0, pad))
            part = part.view(-1, R, case["kv_heads"], case["dim"])
            fresh = part.abs().clone()
            fresh[0, : start % R] = 0
            ids = s["table"][n, first // R:].long()
            scale = _scale64(fresh.amax((1, 3)), TOP[pool])
            if start % R:
                scale[0] = torch.maximum(scale[0], scales[ids[0], :, which])
            scales[ids, :, which] = scale
            part = _round64(part / scale[:, None, :, None], pool) * scale[:, None, :, None]
            val[first:] = part.reshape(-1, case["kv_heads"], case["dim"])[: rows - first]
            held[n] = val.transpose(0, 1)
        out.append(torch.stack(held))
    return {"k": out[0], "v": out[1], "scales": scales}


def _exact_bounds(case, s):
    R = case["page"]
    out = torch.zeros(s["bounds"].shape, dtype=torch.float64, device=s["bounds"].device)
    for n, count in enumerate(s["lengths"].tolist()):
        k = _rows64(s, 0, n, torch.arange(count, device=out.device))
        k = torch.cat((k, k[-1:].expand(-count % R, -1, -1))).view(-1, R, *k.shape[1:])  # the last row again fills a page
        hi, lo = k.amax(1), k.amin(1)
        scale = _scale64(torch.maximum(hi.abs(), lo.abs()).amax(2), 127)[..., None]
        ids = s["table"][n, : len(k)].long()
        out[ids] = torch.stack((torch.ceil(hi / scale) * scale, torch.floor(lo / scale) * scale), 2)
    return {"bounds": out}


def _exact_sparse(case, s):
    N, Hq, T, D = s["q"].shape
    H, R, K, G = case["kv_heads"], case["page"], case["select"], case["group"]
    dev = s["q"].device
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=dev)
    index = torch.full((N, H, T, K), -1, dtype=torch.int32)
    for n, count in enumerate(s["lengths"].tolist()):
        pages = -(-count // R)
        ids = s["table"][n, :pages].long()
        at = torch.arange(count, device=dev)
        k, v = _rows64(s, 0, n, at), _rows64(s, 1, n, at)
        both, scale = s["bounds"][ids].double(), s["bound_scales"][ids].double()
        for h in range(H):
            q = s["q"][n, h * G: (h + 1) * G].double()  # [G, T, D]
            step = _scale64(q.abs().amax((0, 2)), 127)[None, :, None]
            whole = torch.round(q / step)
            best = torch.where(whole[..., None, :] > 0, whole[..., None, :] * both[:, h, 0], whole[..., None, :] * both[:, h, 1])
            best = (best.sum(-1).amax(0) * scale[:, h]).cpu()  # [T, pages]
            for t in range(T):
                w = best[t].tolist()
                keep = sorted(sorted(range(pages), key=lambda i: (-w[i], i))[:K])  # noqa: B023
                index[n, h, t, : len(keep)] = torch.tensor(keep, dtype=torch.int32)
                pick = (torch.tensor(keep, device=dev)[:, None] * R + torch.arange(R, device=dev)).view(-1)
                pick = pick[pick < count]
                out[n, h * G: (h + 1) * G, t] = _softmax_product(q[:, t], k[pick, h], v[pick, h], D)
    return {"index": index, "out": out}


def _exact_books(case, s):
    R, P = case["page"], s["free"].shape[0]
    table, lengths, count = s["table"].tolist(), s["lengths"].tolist(), s["count"].tolist()
    free = s["free"].tolist()
    stack = free[: int(s["free_count"])]
    granted, slots, starts = [], [], [0]
    for n, row in enumerate(table):
        has, end = -(-lengths[n] // R), -(-(lengths[n] + count[n]) // R)
        for p in range(has, end):
            if not 0 <= row[p] < P and stack:
                row[p] = stack.pop()
        placed = 0
        for r in range(lengths[n], lengths[n] + count[n]):
            there = 0 <= row[r // R] < P
            placed += there and placed == r - lengths[n]
            slots.append(row[r // R] * R + r % R if there else -1)
        granted.append(placed)
        starts.append(len(slots))
    slots += [-1] * (s["total"] - len(slots))
    given = [list(row) for row in table]
    for n in reversed(range(len(table))):
        for p in reversed(range(-(-lengths[n] // R), len(table[n]))):
            if 0 <= table[n][p] < P:
                stack.append(table[n][p])
                table[n][p] = -1

    def whole(x, dtype=torch.int32):
        return torch.tensor(x, dtype=dtype)

    # what lies past the top of the stack: the pages that were there before
    return {"granted": whole(granted), "slots": whole(slots, torch.int64), "starts": whole(starts), "given": whole(given),
            "table": whole(table), "free": whole(stack + free[len(stack):]), "free_count": whole([len(stack)])}
