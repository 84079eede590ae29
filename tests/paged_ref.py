"""Plain float64 forms of the paged K/V cache operators and the error bounds their kernels are held to (test
infrastructure): sequence by sequence, row by row through the page table, with none of the package's code."""
import torch


def rows_of(table_row, length, R, pages):
    """(row numbers, page ids, rows in the page) of a sequence's rows whose page is in the pool."""
    length = max(0, min(int(length), table_row.numel() * R))
    at = torch.arange(length, device=table_row.device)
    page = table_row.long()[at // R]
    live = (page >= 0) & (page < pages)
    return at[live], page[live], at[live] % R


def attention(q, k_pages, v_pages, table, lengths, scale, weights=None):
    """(out, weights, out's bound, weights' bound): float64, and how far fp32 arithmetic may be from it.

    Bound of a probability, relative: a score is a sum of D products in fp32, |ds| <= (D + 2) 2^-24 sum |q k| |scale|; its
    scaling to log2 units, the subtraction of the reference and the exponential add three roundings of at most 2^-23 of
    |s| + |m| and 2^-21 of the result; the sums over the keys add a rounding per step of the longest chain, at most
    n / 32 + 128 of them; numerator and normaliser carry it alike, hence twice. bf16 value products take the probabilities
    as two bf16 terms: 2^-16 of each. The result is rounded to the output's type: eps / 2 of it."""
    N, Hq, T, D = q.shape
    P, H, R, _ = k_pages.shape
    out, tol = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    w = None if weights is None else weights.double().clone()
    wtol = None if weights is None else torch.zeros_like(w)
    split = 2.0 ** -16 if q.dtype == torch.bfloat16 else 0.0
    for n in range(N):
        at, page, row = rows_of(table[n], lengths[n], R, P)
        if not len(at):
            continue
        k, v = k_pages[page, :, row].double(), v_pages[page, :, row].double()  # [rows, H, D]
        chain = (len(at) / 32 + 128) * 2.0 ** -24
        for h in range(Hq):
            kh, vh = k[:, h // (Hq // H)], v[:, h // (Hq // H)]
            qh = q[n, h].double()
            s = qh @ kh.t() * scale
            m = s.max(dim=1, keepdim=True).values
            p = torch.where(m == -torch.inf, torch.zeros_like(s), torch.exp(s - m))
            total = p.sum(1, keepdim=True)
            p = torch.where(total == 0, torch.zeros_like(p), p / total)
            finite = torch.where(torch.isfinite(kh), kh, torch.zeros_like(kh)).abs()
            ds = (D + 2) * 2.0 ** -24 * (qh.abs() @ finite.t()) * abs(scale)
            fin = torch.where(torch.isfinite(s), s, torch.zeros_like(s)).abs()
            e = 2 * (ds.max(1).values + 3 * 2.0 ** -23 * fin.max(1).values * 1.4427 + 2.0 ** -21 + chain)[:, None]
            out[n, h] = p @ vh
            tol[n, h] = (p @ vh.abs()) * (e + split) + out[n, h].abs() * torch.finfo(q.dtype).eps / 2
            if w is not None:
                w[n, at] += p.sum(0)
                wtol[n, at] += (p * e).sum(0)
    if w is not None:
        # the sum over heads and rows, then its addition to what is there
        wtol += w.abs() * (Hq * T + 2) * 2.0 ** -24
    # denormal results: fp32 arithmetic of the probabilities flushes below 2^-126
    return out, w, tol + 2.0 ** -100, None if wtol is None else wtol + 2.0 ** -100


def near(got, want, tol, what=""):
    """got within tol of want; NaN where want is NaN."""
    got, want = got.double().cpu(), want.cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    over = torch.where(torch.isnan(want), torch.zeros_like(want), (got - want).abs() / tol.cpu())
    worst = float(over.max()) if over.numel() else 0.0
    print(f"[paged] {what}: {worst:.3f} of the bound", flush=True)
    assert worst <= 1.0, f"{what}: {worst} times the bound"


def append(k_pages, v_pages, table, lengths, k, v, count=None):
    """The pools after an append, as new tensors."""
    kp, vp = k_pages.clone(), v_pages.clone()
    P, H, R, D = kp.shape
    cap = table.shape[1] * R
    for n in range(table.shape[0]):
        start = max(0, min(int(lengths[n]), cap))
        T = k.shape[2] if count is None else max(0, min(int(count[n]), k.shape[2]))
        for t in range(T):
            if start + t >= cap:
                break
            page = int(table[n, (start + t) // R])
            if 0 <= page < P:
                kp[page, :, (start + t) % R] = k[n, :, t]
                vp[page, :, (start + t) % R] = v[n, :, t]
    return kp, vp


def evict(k_pages, v_pages, table, lengths, weights, keep, recent=0):
    """(k_pages, v_pages, index, kept weights, kept lengths) after an eviction, as new tensors; pools [blocks, pages, ..]."""
    kp, vp = k_pages.clone(), v_pages.clone()
    B, P, H, R, D = kp.shape
    N, cap = table.shape[0], table.shape[1] * R
    each = [int(keep)] * N if not torch.is_tensor(keep) else [int(x) for x in keep]
    K = min(int(keep), cap) if not torch.is_tensor(keep) else cap
    index = torch.full((N, K), -1, dtype=torch.int32)
    kw = torch.zeros(N, cap)
    kept = torch.zeros(N, dtype=torch.int32)
    w = torch.where(torch.isnan(weights), torch.full_like(weights, -torch.inf), weights).cpu()
    for n in range(N):
        length = max(0, min(int(lengths[n]), cap))
        c = max(0, min(length, each[n], K))
        last = min(recent, c)
        order = sorted(range(length - last), key=lambda i: (-float(w[n, i]), i))
        held = set(order[:c - last]) | set(range(length - last, length))
        slot = list(range(c))
        tail = [i for i in range(c, length) if i in held]
        for to, back in zip([i for i in range(c) if i not in held], tail):
            slot[to] = back
            pt, pb = int(table[n, to // R]), int(table[n, back // R])
            if 0 <= pt < P and 0 <= pb < P:
                kp[:, pt, :, to % R] = k_pages[:, pb, :, back % R]
                vp[:, pt, :, to % R] = v_pages[:, pb, :, back % R]
        index[n, :c] = torch.tensor(slot, dtype=torch.int32)
        kw[n, :c] = weights[n].cpu()[slot]
        kept[n] = c
    return kp, vp, index, kw, kept
