"""GPU test of random runs over a pool: pages reserved and released on the device, rows appended padded or packed, bounds of what
was appended, attention over all pages and over chosen or listed ones, rows read back, each against the plain forms. Types, head
layouts, page sizes, missing pages, wide tables, pools that are blocks of a larger one and stacks that run dry are drawn."""
import random

import pytest
import torch

import paged8_ref as ref
import paged_ref

pytestmark = pytest.mark.gpu
BF, F32, E4, I8, I32 = torch.bfloat16, torch.float32, torch.float8_e4m3fn, torch.int8, torch.int32


@pytest.mark.parametrize("seed", range(24))
def test_random_runs(dev, seed):
    import tabicl_mi355_paged as paged
    r = random.Random(seed)
    g = torch.Generator(device=dev).manual_seed(seed)
    code = [BF, F32, E4, I8][seed % 4]
    q8 = code in (E4, I8)
    dtype = r.choice([BF, F32]) if q8 else code
    N, H, G, D, R = r.randint(1, 6), r.randint(1, 4), r.choice([1, 1, 2, 5, 16, 20]), r.choice([32, 64, 128]), r.choice([16, 32, 64, 128])
    M = r.choice([1, 2, 5, 9, 40])
    P = max(1, int(N * M * r.choice([0.3, 0.8, 1.2])))
    blocks = r.randint(1, 3)
    mine = r.randrange(blocks)

    def pool():
        x = torch.zeros(P, blocks, H, R, D, device=dev).to(code)
        return x[:, mine]

    kp, vp = pool(), pool()
    scales = torch.full((P, H, 2), float("nan"), device=dev) if q8 else None  # nobody has written them
    wide = torch.full((N, M + r.randint(0, 3)), -1, dtype=I32, device=dev)
    table = wide[:, :M]
    free = torch.randperm(P, generator=g, device=dev).to(I32)
    fc = torch.tensor([P], dtype=I32, device=dev)
    n = torch.zeros(N, dtype=I32, device=dev)
    bnd, bs = torch.zeros(P, H, 2, D, dtype=I8, device=dev), torch.zeros(P, H, device=dev)
    books = ref.Books(table.tolist(), free.tolist(), P, P, R)
    wk, wv, ws = kp.cpu(), vp.cpu(), scales.cpu() if q8 else None
    print(f"[random] seed {seed} {code} {dtype} N {N} H {H} G {G} D {D} R {R} M {M} P {P} block {mine} of {blocks}", flush=True)
    for turn in range(4):
        most = r.choice([1, 3, R, 2 * R + 3, 5 * R])
        new = [r.choice([0, 1, most, r.randint(0, most)]) for _ in range(N)]
        count = torch.tensor(new, dtype=I32, device=dev)
        granted = paged.paged_reserve(table, n, count, free, fc, R)
        assert granted.tolist() == books.reserve(n.tolist(), new)
        T = max(1, max(new))
        k, v = (torch.randn(N, T, H, D, generator=g, device=dev).mul(2.0 ** r.randint(-3, 3)).to(dtype).transpose(1, 2) for _ in range(2))
        if r.random() < 0.5:
            pick = [torch.cat([x[i, :, :new[i]].transpose(0, 1) for i in range(N)] + [x[0, :, :1].transpose(0, 1)]) for x in (k, v)]
            total = sum(new) + 1  # one row of no request
            slots, starts = paged.paged_slots(table, n, count, total, P, R)
            s, st = books.slots(n.tolist(), new, total)
            assert slots.tolist() == s and starts.tolist() == st
            paged.paged_append_packed(kp, vp, table, n, count, *pick, slots, starts, scales)
        else:
            paged.paged_append(kp, vp, table, n, k, v, count, scales)
        t = torch.tensor(books.table, dtype=I32)
        lengths = n.tolist()
        if q8:
            wk, wv, ws = (x.to(code) if i < 2 else x for i, x in
                          enumerate(ref.append(wk, wv, ws, t, lengths, k.cpu(), v.cpu(), new)))
            live = ws == ws
            assert torch.equal(torch.isnan(scales.cpu()), ~live) and torch.equal(scales.cpu()[live], ws[live])
        else:
            wk, wv = paged_ref.append(wk, wv, t, torch.tensor(lengths), k.cpu(), v.cpu(), torch.tensor(new))
        assert torch.equal(kp.cpu().contiguous().view(torch.uint8), wk.contiguous().view(torch.uint8))
        assert torch.equal(vp.cpu().contiguous().view(torch.uint8), wv.contiguous().view(torch.uint8))
        before = n.clone()
        n += granted
        if r.random() < 0.5:
            paged.paged_bounds(kp, table, n, bnd, bs, before, most, scales)
        else:
            paged.paged_bounds(kp, table, n, bnd, bs, scales=scales)
        kk, vv = (ref.values(w, ws, i) if q8 else w.double() for i, w in enumerate((wk, wv)))
        for (page, h), (hi, lo, step) in ref.bounds(kk, t, n.tolist()).items():
            assert torch.equal(bnd[page, h].double().cpu(), torch.stack((hi, lo))) and float(bs[page, h]) == step
        Tq, K = r.choice([1, 2, 7, 17, 40]), r.randint(1, M + 1)
        q = (torch.randn(N, H * G, Tq, D, generator=g, device=dev) * r.choice([0.3, 2.0])).to(dtype)
        sc = D ** -0.5
        out = paged.paged_attention(q, kp, vp, table, n, scales=scales)
        want, _, tol, _ = paged_ref.attention(q.cpu(), kk, vv, t, n.tolist(), sc)
        paged_ref.near(out, want, tol, f"all pages, turn {turn}")
        index = paged.paged_select(q, bnd, bs, table, n, R, K)
        assert torch.equal(index.cpu(), ref.select(q, bnd, bs, t, n.tolist(), R, K))
        any_ = torch.randint(-2, M + 2, index.shape, generator=g, device=dev, dtype=I32)
        for what, x in (("chosen", index), ("listed", any_)):
            few = paged.paged_sparse_attention(q, kp, vp, table, n, x, scales=scales)
            want, tol = ref.sparse_attention(q.cpu(), kk, vv, t, n.tolist(), x.cpu(), sc)
            paged_ref.near(few, want, tol, f"{what}, turn {turn}")
        rows = r.randint(1, M * R)
        gk, gv = paged.paged_gather(kp, vp, table, n, rows, scales, F32 if q8 else None)
        for i, length in enumerate(n.tolist()):
            at, page, row = paged_ref.rows_of(t[i], min(length, rows), R, P)
            for got, w in ((gk, kk), (gv, vv)):
                assert torch.equal(got[i, :, at].double().cpu(), w[page, :, row].transpose(0, 1))
        n.copy_(torch.tensor([r.choice([0, x, x, r.randint(0, x)]) for x in n.tolist()], dtype=I32))
        paged.paged_release(table, n, free, fc, R)
        books.release(n.tolist())
        assert table.tolist() == books.table and int(fc) == len(books.stack) and free[:int(fc)].tolist() == books.stack
        assert (wide[:, M:] == -1).all()


@pytest.mark.parametrize("dtype", [BF, I8], ids=["bf16", "int8"])
def test_cache_of_no_more_rows_than_the_selection(dev, dtype):
    # valid_kv_len within the selected pages: attention over all of those rows
    import tabicl_mi355_paged as paged
    g = torch.Generator(device=dev).manual_seed(6)
    S, H, D, R, K = 3, 8, 64, 16, 4
    c = paged.PagedIclKVCache(S, 1, H, D, 600, 90, R, dtype, dev, select=K)
    k, v = (torch.randn(S, H, 321, D, generator=g, device=dev).to(BF) for _ in range(2))
    c.append(0, k, v, [321, 51, 0])
    kk, vv = (ref.values(x, c.scales[0], i) if c.scales is not None else x.double() for i, x in enumerate((c.keys[0], c.values[0])))
    q = torch.randn(S, H, 3, D, generator=g, device=dev).to(BF)
    for most in (K * R, K * R - 5, 1, 0, torch.tensor([K * R, 7, 3], device=dev), torch.tensor(K * R, device=dev)):
        out = c.query(0, q, most)
        least = torch.as_tensor(most, device=dev).expand(S).clamp(max=10 ** 6).int()
        want, _, tol, _ = paged_ref.attention(q, kk, vv, c.table, torch.minimum(c.lengths[0], least), D ** -0.5)
        paged_ref.near(out, want, tol, f"at most {most}")
