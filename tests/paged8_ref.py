"""Plain forms of the 8-bit paged cache, of the selection of pages and of the books of a pool (test infrastructure): row by
row and page by page on the CPU, in float64 and whole numbers, with none of the package's code."""
import math

import torch

import paged_ref

TOP = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}
LOW, HIGH = -60, 100  # the exponents of a scale


def exponent(most, top):
    """The smallest k in [LOW, HIGH] with most <= top 2^k."""
    k = LOW
    while k < HIGH and most > top * 2.0 ** k:
        k += 1
    return k


def codes(x, dtype):
    """float64 values to the nearest code (ties to even), as float64; NaN stays NaN in e4m3 and is 0 in int8."""
    if dtype is torch.int8:
        return torch.nan_to_num(x, nan=0.0, posinf=127.0, neginf=-127.0).round().clamp(-127, 127)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(2.0 ** -6, 448.0))) - 3)  # 4 significant bits, 2^-9 at least
    return ((x / step).round() * step).clamp(-448, 448)


def values(pages, scales, which):
    """The float64 values of K (0) or V (1) pages."""
    return pages.float().double() * scales[:, :, which, None, None].double()


def append(k_pages, v_pages, scales, table, lengths, k, v, count=None, starts=None):
    """The pools (as float64 codes) and the scales after an append. k, v [N, H, T, D], or packed [total, H, D] with starts."""
    dtype = k_pages.dtype
    scales = scales.clone()
    P, H, R, D = k_pages.shape
    cap = table.shape[1] * R
    out = []
    for which, pages, x in ((0, k_pages, k), (1, v_pages, v)):
        pages = pages.float().double()
        for n in range(table.shape[0]):
            start = max(0, min(int(lengths[n]), cap))
            if starts is None:
                rows = x[n].transpose(0, 1).double()  # [T, H, D]
                T = rows.shape[0] if count is None else max(0, min(int(count[n]), rows.shape[0]))
            else:
                rows = x[int(starts[n]):].double()
                T = max(0, min(int(count[n]), rows.shape[0]))
            end = min(start + T, cap)
            for p in range(start // R, -(-end // R)):
                lo, hi = max(start, p * R), min(end, (p + 1) * R)
                page = int(table[n, p])
                if lo >= hi or not 0 <= page < P:
                    continue
                for h in range(H):
                    new = rows[lo - start:hi - start, h]
                    finite = new[torch.isfinite(new)].abs()
                    s = 2.0 ** exponent(float(finite.max()) if finite.numel() else 0.0, TOP[dtype])
                    held = lo - p * R
                    old = float(scales[page, h, which])
                    if held and old > s:
                        s = old
                    if held and s != old:
                        pages[page, h, :held] = codes(pages[page, h, :held] * (old / s), dtype)
                    pages[page, h, held:held + hi - lo] = codes(new / s, dtype)
                    scales[page, h, which] = s
        out.append(pages)
    return out[0], out[1], scales


def bounds(k, table, lengths, start=None, rows=None):
    """{(page, h): (hi, lo, scale)} as whole numbers and a power of two, over float64 keys k [pages, H, R, D]."""
    P, H, R, D = k.shape
    out = {}
    for n in range(table.shape[0]):
        length = max(0, min(int(lengths[n]), table.shape[1] * R))
        first = max(0, int(start[n])) // R if start is not None else 0
        for p in range(first, -(-length // R)):
            page = int(table[n, p])
            if not 0 <= page < P:
                continue
            for h in range(H):
                x = k[page, h, :min(R, length - p * R)]
                none = torch.isnan(x).all(0)
                hi = torch.where(torch.isnan(x), -math.inf, x).amax(0)
                lo = torch.where(torch.isnan(x), math.inf, x).amin(0)
                hi, lo = torch.where(none, 0.0, hi), torch.where(none, 0.0, lo)
                both = torch.cat((hi, lo))
                finite = both[torch.isfinite(both)].abs()
                s = 2.0 ** exponent(float(finite.max()) if finite.numel() else 0.0, 127.0)
                out[page, h] = (torch.ceil(hi / s).clamp(-127, 127), torch.floor(lo / s).clamp(-127, 127), s)
    return out


def select(q, bnd, bound_scales, table, lengths, R, K):
    """index [N, H, T, K] from bounds [pages, H, 2, D] (whole numbers)."""
    N, Hq, T, D = q.shape
    P, H = bnd.shape[:2]
    G = Hq // H
    index = torch.full((N, H, T, K), -1, dtype=torch.int32)
    q, bnd, bound_scales = q.double().cpu(), bnd.double().cpu(), bound_scales.double().cpu()
    for n in range(N):
        length = max(0, min(int(lengths[n]), table.shape[1] * R))
        pages = [p for p in range(-(-length // R)) if 0 <= int(table[n, p]) < P]
        if not pages:
            continue
        ids = table[n, pages].long().cpu()
        for h in range(H):
            for t in range(T):
                rows = q[n, h * G:(h + 1) * G, t]
                finite = rows[torch.isfinite(rows)].abs()
                step = 2.0 ** exponent(float(finite.max()) if finite.numel() else 0.0, 127.0)
                u = torch.nan_to_num(rows / step, nan=0.0, posinf=127.0, neginf=-127.0).round().clamp(-127, 127)  # [G, D]
                hi, lo = bnd[ids, h, 0], bnd[ids, h, 1]  # [pages, D]
                # the larger of u hi and u lo, as long as hi >= lo
                best = torch.where(u[:, None] > 0, u[:, None] * hi, u[:, None] * lo).sum(-1).amax(0) * bound_scales[ids, h]
                order = sorted(range(len(pages)), key=lambda i: (-float(best[i]), i))[:K]  # noqa: B023
                keep = sorted(pages[i] for i in order)
                index[n, h, t, :len(keep)] = torch.tensor(keep, dtype=torch.int32)
    return index


def sparse_attention(q, k, v, table, lengths, index, scale):
    """(out, bound) of paged_ref.attention over the listed pages; k, v float64 pools (or bf16 / fp32 ones)."""
    N, Hq, T, D = q.shape
    P, H, R, _ = k.shape
    G = Hq // H
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol = torch.full_like(out, 2.0 ** -100)
    for n in range(N):
        length = max(0, min(int(lengths[n]), table.shape[1] * R))
        for h in range(H):
            for t in range(T):
                ids, live = [], []
                for p in index[n, h, t].tolist():
                    if 0 <= p < table.shape[1] and p * R < length:
                        ids.append(int(table[n, p]))
                        live.append(min(R, length - p * R))
                # one page each: the listed pages as a table of their own, full pages first
                order = sorted(range(len(ids)), key=lambda i: -live[i])
                rows_k = [k[ids[i], h, :live[i]] for i in order if 0 <= ids[i] < P]
                rows_v = [v[ids[i], h, :live[i]] for i in order if 0 <= ids[i] < P]
                if not rows_k:
                    continue
                kk, vv = torch.cat(rows_k), torch.cat(rows_v)
                L = len(kk)
                one = torch.arange(1, dtype=torch.int32, device=q.device).view(1, 1)
                o, _, b, _ = paged_ref.attention(q[n:n + 1, h * G:(h + 1) * G, t:t + 1], kk.view(1, 1, L, D), vv.view(1, 1, L, D),
                                                 one, torch.tensor([L]), scale)
                out[n, h * G:(h + 1) * G, t], tol[n, h * G:(h + 1) * G, t] = o[0, :, 0], b[0, :, 0]
    return out, tol


class Books:
    """A pool's books in Python lists."""

    def __init__(self, table, free, free_count, pages, R):
        self.table = [list(map(int, r)) for r in table]
        self.stack = list(map(int, free))[:max(0, min(int(free_count), pages))]
        self.pages, self.R = pages, R

    def has(self, page):
        return 0 <= page < self.pages

    def _span(self, n, length, add):
        M = len(self.table[n])
        length = max(0, min(int(length), M * self.R))
        add = max(0, int(add))
        return length, add, range(-(-length // self.R), min(M, -(-(length + add) // self.R)))

    def reserve(self, lengths, count):
        granted = []
        for n, row in enumerate(self.table):
            length, add, span = self._span(n, lengths[n], count[n])
            for p in span:
                if not self.has(row[p]) and self.stack:
                    row[p] = self.stack.pop()
            first = next((p for p in range(length // self.R, span.stop) if not self.has(row[p])), len(row))
            granted.append(max(0, min(add, first * self.R - length)))
        return granted

    def slots(self, lengths, count, total):
        out, starts = [], [0]
        for n, row in enumerate(self.table):
            length = max(0, int(lengths[n]))
            for t in range(max(0, int(count[n]))):
                p, r = divmod(length + t, self.R)
                out.append(row[p] * self.R + r if p < len(row) and self.has(row[p]) else -1)
            starts.append(len(out))
        return (out + [-1] * total)[:total], starts

    def release(self, lengths):
        for n in reversed(range(len(self.table))):
            row = self.table[n]
            keep = -(-max(0, min(int(lengths[n]), len(row) * self.R)) // self.R)
            for p in reversed(range(keep, len(row))):
                if self.has(row[p]):
                    if len(self.stack) < self.pages:
                        self.stack.append(row[p])
                    row[p] = -1
