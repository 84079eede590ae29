"""The operators of the paged K/V cache as timed cases: attention of one or a few new rows over the cache, the same
with the attention weights added up per cached row, rows written into the pages, and eviction by those weights.

listed() names the cases; draw(rng) gives another one of the same ranges; prepare / run / work take a case. Where
`own` is false, run() computes an operator from elementary torch operations in fp32; where it is true, it calls the
package. exact() restates a case in float64, sequence by sequence. Inputs come from torch's device generator and the
seed alone.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tabiclv2-torchtpu-v5p-benchmark_amd")
DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
ES = {"bf16": 2, "fp32": 4}
HEADS, DIM = 8, 64  # the ICL stage


def _paged():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import tabicl_mi355_paged
    return tabicl_mi355_paged


# ---------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------
def _attn(name, seqs, shortest, longest, rows, dtype="bf16", kv_heads=HEADS, group=1, dim=DIM, page=64, weights=False):
    return {"name": name, "kind": "attn", "seqs": seqs, "shortest": shortest, "longest": longest, "rows": rows,
            "dtype": dtype, "kv_heads": kv_heads, "group": group, "dim": dim, "page": page, "weights": weights}


def listed() -> list:
    return [
        # one test row of a small table, 8 estimators, as a service answers it (latency)
        _attn("attn_one_small", 8, 700, 700, 1),
        # one test row at the headline table: 45,000 cached train rows
        _attn("attn_one_large", 8, 45000, 45000, 1),
        # a mixed batch: 64 tables of 500 to 10,000 train rows, 4 test rows each
        _attn("attn_ragged", 64, 500, 10000, 4),
        # a block of 64 test rows over 5,000 train rows
        _attn("attn_block", 8, 5000, 5000, 64),
        # fp32 validation mode, small pages, odd lengths
        _attn("attn_fp32", 4, 9001, 12345, 3, dtype="fp32", page=16),
        # grouped heads of 128 dims, a batch of 16 with one new row each
        _attn("attn_grouped", 16, 1111, 8192, 1, group=4, dim=128, page=32),
        # attention that also adds up the weights: one row over a small cache, 16 rows over the headline one
        _attn("weights_small", 8, 1999, 1999, 1, weights=True),
        _attn("weights_large", 8, 45000, 45000, 16, weights=True),
        # one new row per sequence written into the cache; a block's train rows at fit time
        {"name": "append_one", "kind": "append", "seqs": 8, "start": 1000, "rows": 1, "dtype": "bf16",
         "kv_heads": HEADS, "dim": DIM, "page": 64},
        {"name": "append_fit", "kind": "append", "seqs": 8, "start": 0, "rows": 45000, "dtype": "bf16",
         "kv_heads": HEADS, "dim": DIM, "page": 64},
        # a small cache cut to half over the 12 ICL blocks; a larger one cut to 10,000 rows
        {"name": "evict_small", "kind": "evict", "seqs": 8, "shortest": 1000, "longest": 1000, "keep": 512,
         "recent": 32, "blocks": 12, "dtype": "bf16", "kv_heads": HEADS, "dim": DIM, "page": 64},
        {"name": "evict_large", "kind": "evict", "seqs": 8, "shortest": 16384, "longest": 16384, "keep": 10000,
         "recent": 100, "blocks": 4, "dtype": "bf16", "kv_heads": HEADS, "dim": DIM, "page": 64},
    ]


def _log(rng, lo: int, hi: int) -> int:
    """An integer spread evenly over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    kind = rng.choice(["attn", "attn", "attn", "weights", "weights", "append", "evict"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    kv_heads, dim = rng.choice([(8, 64), (8, 64), (4, 32), (8, 32), (8, 128), (2, 128)])
    case = {"kind": kind, "dtype": dtype, "kv_heads": kv_heads, "dim": dim, "page": rng.choice([16, 32, 64, 128, 256])}
    row = kv_heads * dim * ES[dtype] * 2  # bytes of one cached row, K and V
    seqs = _log(rng, 1, 64)
    if kind in ("attn", "weights"):
        longest = _log(rng, 1, max(1, min(50000, 700000000 // (seqs * row))))
        group = rng.choice([1, 1, 2, 4])
        most = 46000000 // (seqs * kv_heads * group * longest)
        return {**case, "kind": "attn", "seqs": seqs, "shortest": max(1, int(longest * rng.choice([1.0, rng.random()]))),
                "longest": longest, "rows": _log(rng, 1, max(1, min(64, most))), "group": group,
                "weights": kind == "weights"}
    if kind == "append":
        rows = _log(rng, 1, max(1, min(50000, 350000000 // (seqs * row))))
        return {**case, "seqs": seqs, "start": rng.choice([0, rng.randint(1, 2000)]), "rows": rows}
    blocks = rng.choice([1, 2, 12])
    longest = _log(rng, 20, max(20, min(50000, 700000000 // (seqs * row * blocks))))
    keep = max(1, int(longest * rng.uniform(0.2, 0.95)))
    return {**case, "seqs": seqs, "shortest": max(1, int(longest * rng.choice([1.0, rng.random()]))), "longest": longest,
            "keep": keep, "recent": rng.choice([0, keep // 16]), "blocks": blocks}


def _lengths(case) -> list:
    """The sequences' lengths, spread evenly over the logarithm from the shortest to the longest."""
    lo, hi, n = case["shortest"], case["longest"], case["seqs"]
    return [round(lo * (hi / lo) ** (i / (n - 1))) if n > 1 else hi for i in range(n)]


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def prepare(case, seed: int) -> dict:
    """Pages in random order behind a page table, as a cache that has been in use for a while holds them. Heads differ in
    sharpness, so that some rows of the cache draw far more weight than others."""
    dev = torch.device("cuda", 0)
    g = torch.Generator(device=dev).manual_seed(1000003 * (seed + 1))
    dt, R, H, D, N = DT[case["dtype"]], case["page"], case["kv_heads"], case["dim"], case["seqs"]

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device=dev, dtype=dtype)

    if case["kind"] == "append":
        held = [case["start"]] * N
        total = [case["start"] + case["rows"]] * N
    else:
        order = torch.randperm(N, generator=g, device=dev).tolist()
        held = [_lengths(case)[i] for i in order]
        total = held
    width = -(-max(total) // R)
    ids = torch.randperm(N * width + 3, generator=g, device=dev)[: N * width].to(torch.int32)
    blocks = (case["blocks"],) if case["kind"] == "evict" else ()
    s = {"case": case, "table": ids.view(N, width), "lengths": torch.tensor(held, dtype=torch.int32, device=dev),
         "k_pages": randn(*blocks, N * width + 3, H, R, D, dtype=dt),
         "v_pages": randn(*blocks, N * width + 3, H, R, D, dtype=dt)}
    if case["kind"] == "append":
        # heads read out of a K|V projection [N, T, 2, H, D]
        kv = randn(N, case["rows"], 2, H, D, dtype=dt)
        s["k"], s["v"] = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
    elif case["kind"] == "attn":
        q = randn(N, H * case["group"], case["rows"], D) * torch.exp(randn(N, H * case["group"], 1, 1) * 0.5)
        s["q"] = q.to(dt)
        s["weights"] = torch.rand(N, width * R, generator=g, device=dev) if case["weights"] else None
    else:
        # what a few hundred queries add up to: log-normal, a tenth of the rows never drew any weight
        w = torch.exp(randn(N, width * R) * 1.5 - 4.0)
        s["weights"] = torch.where(torch.rand(N, width * R, generator=g, device=dev) < 0.1, torch.zeros_like(w), w)
    return s


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(s):
    return {"attn": _run_attn, "append": _run_append, "evict": _run_evict}[s["case"]["kind"]](s)


def _run_attn(s):
    q, kp, vp, table, lengths, weights = s["q"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], s["weights"]
    if own:
        out = _paged().paged_attention(q, kp, vp, table, lengths, weights)
        return {"out": out} if weights is None else {"out": out, "weights": weights}
    N, Hq, T, D = q.shape
    H, R = kp.shape[1], kp.shape[2]
    L = table.shape[1] * R
    rows = table.long()
    k = kp[rows].float().permute(0, 2, 1, 3, 4).reshape(N, H, L, D)
    v = vp[rows].float().permute(0, 2, 1, 3, 4).reshape(N, H, L, D)
    live = (torch.arange(L, device=q.device) < lengths[:, None]).view(N, 1, 1, L)
    scores = torch.matmul(q.float().reshape(N, H, -1, D), k.transpose(2, 3)) * D ** -0.5
    scores = torch.where(live, scores, -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    out = torch.matmul(p, v).view(N, Hq, T, D).to(q.dtype)
    if weights is None:
        return {"out": out}
    weights += p.sum((1, 2))
    return {"out": out, "weights": weights}


def _run_append(s):
    kp, vp, table, lengths, k, v = s["k_pages"], s["v_pages"], s["table"], s["lengths"], s["k"], s["v"]
    if own:
        _paged().paged_append(kp, vp, table, lengths, k, v)
        return {"k_pages": kp, "v_pages": vp}
    R = kp.shape[2]
    at = lengths.long()[:, None] + torch.arange(k.shape[2], device=k.device)
    page, row = table.long().gather(1, at // R), at % R
    kp[page, :, row] = k.transpose(1, 2)
    vp[page, :, row] = v.transpose(1, 2)
    return {"k_pages": kp, "v_pages": vp}


def _run_evict(s):
    kp, vp, table, lengths, weights, c = s["k_pages"], s["v_pages"], s["table"], s["lengths"], s["weights"], s["case"]
    if own:
        index, kept_weights, kept = _paged().paged_evict(kp, vp, table, lengths, weights, c["keep"], c["recent"])
        return {"k_pages": kp, "v_pages": vp, "index": index, "weights": kept_weights, "lengths": kept}
    N, L, R = weights.shape[0], weights.shape[1], kp.shape[3]
    pos = torch.arange(L, device=weights.device).expand(N, L)
    n = lengths.long()[:, None]
    kept = n.clamp(max=c["keep"])
    recent = kept.clamp(max=c["recent"])
    # the most recent rows before all others, rows past the end behind them; ties to the lowest row
    rank_by = torch.where(pos >= n - recent, math.inf, weights)
    rank_by = torch.where(pos >= n, -math.inf, rank_by)
    order = torch.sort(rank_by, dim=1, descending=True, stable=True).indices
    keep = torch.zeros(N, L, dtype=torch.bool, device=weights.device).scatter_(1, order, pos < kept)
    # the i-th place below `kept` that is not kept takes the i-th kept row at or past it
    hole, tail = (pos < kept) & ~keep, (pos >= kept) & keep
    seq, to = hole.nonzero(as_tuple=True)
    _, back = tail.nonzero(as_tuple=True)
    index = torch.where(pos < kept, pos, -1)
    index[seq, to] = back
    index = index[:, : min(c["keep"], L)]
    rows = table.long()
    to_page, to_row, page, row = rows[seq, to // R], to % R, rows[seq, back // R], back % R
    kp[:, to_page, :, to_row] = kp[:, page, :, row]
    vp[:, to_page, :, to_row] = vp[:, page, :, row]
    kept_weights = torch.zeros_like(weights)
    kept_weights[:, : index.shape[1]] = torch.where(index >= 0, weights.gather(1, index.clamp(min=0)), 0.0)
    return {"k_pages": kp, "v_pages": vp, "index": index.int(), "weights": kept_weights, "lengths": kept[:, 0].int()}


def work(case) -> dict:
    """Each input read once and each output written once; for eviction, the rows that have to move (as many as a choice
    without regard to the place leaves below the cut)."""
    es, row = ES[case["dtype"]], case["kv_heads"] * case["dim"] * ES[case["dtype"]] * 2
    if case["kind"] == "append":
        return {"bytes": 2 * case["seqs"] * case["rows"] * row, "flops": 0}
    total = sum(_lengths(case))
    if case["kind"] == "attn":
        heads = case["kv_heads"] * case["group"]
        return {"bytes": total * row + 2 * case["seqs"] * heads * case["rows"] * case["dim"] * es
                + (8 * total if case["weights"] else 0),
                "flops": 4 * total * heads * case["rows"] * case["dim"]}
    moved = kept = 0.0
    for n in _lengths(case):
        k = min(n, case["keep"])
        recent = min(k, case["recent"])
        free = n - recent
        kept += k
        moved += min(k, free) * (1 - (k - recent) / free) if free else 0.0
    return {"bytes": 2 * moved * row * case["blocks"] + 4 * total + 8 * kept, "flops": 0}


# ---------------------------------------------------------------------------------------------
# float64
# ---------------------------------------------------------------------------------------------
def exact(case, seed: int):
    s = prepare(case, seed)
    R = case["page"]
    if case["kind"] == "append":
        for n in range(case["seqs"]):
            at = torch.arange(case["start"], case["start"] + case["rows"], device=s["k"].device)
            flat = s["table"][n].long()[at // R] * R + at % R
            for pages, new in ((s["k_pages"], s["k"]), (s["v_pages"], s["v"])):
                P, H, _, D = pages.shape
                line = pages.transpose(1, 2).reshape(P * R, H, D)
                line[flat] = new[n].transpose(0, 1)
                pages.copy_(line.view(P, R, H, D).transpose(1, 2))
        return {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    if case["kind"] == "attn":
        return _exact_attn(case, s)
    return _exact_evict(case, s)


def _cached(pages, table, n, count, R):
    at = torch.arange(count, device=pages.device)
    return pages[table[n].long()[at // R], :, at % R].double()  # [count, H, D]


def _exact_attn(case, s):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    weights = None if s["weights"] is None else s["weights"].double()
    for n, count in enumerate(s["lengths"].tolist()):
        k = _cached(s["k_pages"], s["table"], n, count, case["page"])
        v = _cached(s["v_pages"], s["table"], n, count, case["page"])
        for h in range(s["q"].shape[1]):
            kh = k[:, h // case["group"]]
            p = torch.softmax(s["q"][n, h].double() @ kh.t() / math.sqrt(case["dim"]), dim=-1)
            out[n, h] = p @ v[:, h // case["group"]]
            if weights is not None:
                weights[n, :count] += p.sum(0)
    return {"out": out} if weights is None else {"out": out, "weights": weights}


def _exact_evict(case, s):
    R, L = case["page"], s["weights"].shape[1]
    index = torch.full((case["seqs"], min(case["keep"], L)), -1, dtype=torch.int32)
    kept_weights = torch.zeros(s["weights"].shape, dtype=torch.float64)
    weights, kept = s["weights"].cpu(), []
    for n, count in enumerate(s["lengths"].tolist()):
        k = min(count, case["keep"])
        recent = min(case["recent"], k)
        w = weights[n].tolist()
        best = sorted(range(count - recent), key=lambda i: (-w[i], i))[: k - recent]
        keep = set(best) | set(range(count - recent, count))
        holes = [i for i in range(k) if i not in keep]
        tail = [i for i in range(k, count) if i in keep]
        slot = list(range(k))
        for to, back in zip(holes, tail):
            slot[to] = back
        index[n, :k] = torch.tensor(slot, dtype=torch.int32)
        kept_weights[n, :k] = weights[n][slot].double()
        kept.append(k)
        if not holes:
            continue
        t = s["table"][n].long()
        to, back = torch.tensor(holes, device=t.device), torch.tensor(tail, device=t.device)
        for pages in (s["k_pages"], s["v_pages"]):
            for b in range(case["blocks"]):
                pages[b, t[to // R], :, to % R] = pages[b, t[back // R], :, back % R]
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"], "index": index, "weights": kept_weights,
            "lengths": torch.tensor(kept, dtype=torch.int32)}
