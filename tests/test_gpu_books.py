"""GPU tests of a pool's books on the device against Python lists (paged8_ref.Books): pages for new rows from the stack, back
to it, the slots of packed rows, the rows into them, and a captured step of a service that is replayed while its requests
grow. Everything is a whole number or a copy, and compared exactly."""
import pytest
import torch

import paged8_ref as ref
import paged_ref

pytestmark = pytest.mark.gpu
BF, F32, E4, I8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn, torch.int8
I32 = torch.int32


def _books(dev, seed, lengths, M, R, spare=5, lost=0):
    """A table whose requests hold pages for `lengths` rows, the other pages on the stack but for `lost` of them."""
    g = torch.Generator().manual_seed(seed)
    N = len(lengths)
    need = [min(M, -(-max(0, n) // R)) for n in lengths]
    P = sum(need) + spare + lost
    ids = torch.randperm(P, generator=g).tolist()
    table = torch.full((N, M), -1, dtype=I32)
    for n in range(N):
        for p in range(need[n]):
            table[n, p] = ids.pop()
    free = torch.zeros(P, dtype=I32)
    stack = ids[:len(ids) - lost]
    free[:len(stack)] = torch.tensor(stack, dtype=I32)
    return table.to(dev), torch.tensor(lengths, dtype=I32, device=dev), free.to(dev), torch.tensor([len(stack)], dtype=I32, device=dev), g


def _same(b, table, free, free_count, what):
    assert table.tolist() == b.table, what
    assert int(free_count) == len(b.stack), what
    assert free[:len(b.stack)].tolist() == b.stack, what


def _step(table, n, count, free, free_count, R, total=None, what=""):
    import tabicl_mi355_paged as paged
    P = free.numel()
    b = ref.Books(table.tolist(), free.tolist(), int(free_count), P, R)
    keep = n.clone(), count.clone(), free.clone()
    print(f"[books] {what} table {tuple(table.shape)} R {R} pages {P}", flush=True)
    granted = paged.paged_reserve(table, n, count, free, free_count, R)
    want = b.reserve(n.tolist(), count.tolist())
    _same(b, table, free, free_count, what)
    assert granted.tolist() == want, what
    total = sum(max(0, c) for c in count.tolist()) + 3 if total is None else total
    slots, starts = paged.paged_slots(table, n, count, total, P, R)
    ws, wst = b.slots(n.tolist(), count.tolist(), total)
    assert slots.dtype == torch.int64 and slots.tolist() == ws and starts.tolist() == wst, what
    for t, k in zip((n, count, free), keep):
        assert torch.equal(t, k)
    return b


@pytest.mark.parametrize("R", [16, 64, 1024])
def test_reserve_slots_release(dev, R):
    import tabicl_mi355_paged as paged
    lengths = [0, 1, R - 1, R, R + 1, 3 * R, 5 * R - 2, 0]
    counts = [0, 1, 1, 1, 2 * R, 0, 3, 7 * R + 5]
    table, n, free, fc, g = _books(dev, R, lengths, 9, R, spare=40)
    count = torch.tensor(counts, dtype=I32, device=dev)
    before = table.clone(), free.clone(), fc.clone()
    b = _step(table, n, count, free, fc, R, what="room for all")
    # the release of what was reserved restores the books
    paged.paged_release(table, n, free, fc, R)
    for t, w in zip((table, free, fc), before):
        assert torch.equal(t, w)
    b.release(n.tolist())
    _same(b, table, free, fc, "released")
    # then everything back
    zero = torch.zeros_like(n)
    b.release(zero.tolist())
    paged.paged_release(table, zero, free, fc, R)
    _same(b, table, free, fc, "all back")
    assert (table == -1).all()


@pytest.mark.parametrize("spare", [0, 1, 3, 11])
def test_too_few_pages(dev, spare):
    table, n, free, fc, g = _books(dev, spare, [5, 30, 0, 64, 17], 8, 16, spare=spare, lost=2)
    count = torch.tensor([40, 2, 100, 1, 90], dtype=I32, device=dev)
    _step(table, n, count, free, fc, 16, what="too few")
    _step(table, n, count, free, fc, 16, what="again")  # nothing left, or what was missing


def test_odd_books(dev):
    # lengths and counts below 0, past the table, entries that are no pages, pages in place behind the rows, a full table
    table, n, free, fc, g = _books(dev, 3, [5, 30, 0, 64, 17, 128], 8, 16, spare=30)
    n[:] = torch.tensor([-5, 30, 2 ** 31 - 1, 100, 17, 128], dtype=I32)
    count = torch.tensor([20, -3, 5, 1000, 0, 1], dtype=I32, device=dev)
    table[3, 7] = free[0]  # reserved earlier
    free[:29] = free[1:30].clone()
    fc -= 1
    table[0, 0], table[0, 1], table[4, 0] = 2 ** 31 - 1, -7, free.numel()
    b = _step(table, n, count, free, fc, 16, what="odd")
    import tabicl_mi355_paged as paged
    n[:] = torch.tensor([-5, 1, 2 ** 31 - 1, 100, 17, 16], dtype=I32)
    b.release(n.tolist())
    paged.paged_release(table, n, free, fc, 16)
    _same(b, table, free, fc, "odd release")
    fc[0] = 2 ** 31 - 1  # more than there can be
    b = _step(table, torch.zeros_like(n), torch.full_like(n, 300), free, fc, 16, what="a stack that claims too much")
    fc[0] = -9
    _step(table, torch.zeros_like(n), torch.full_like(n, 300), free, fc, 16, what="an empty one")


@pytest.mark.parametrize("N,most", [(1, 5000), (3, 0), (300, 40), (1023, 3), (1025, 9), (5000, 2), (2048, 70), (70, 16000)])
def test_many_requests(dev, N, most):
    import tabicl_mi355_paged as paged
    g = torch.Generator().manual_seed(N)
    lengths = torch.randint(0, 50, (N,), generator=g).tolist()
    M = (50 + most) // 16 + 2
    table, n, free, fc, _ = _books(dev, N, lengths, M, 16, spare=N * M // 2)
    count = torch.randint(0, most + 1, (N,), generator=g).to(I32).to(dev)
    b = _step(table, n, count, free, fc, 16, what="many")
    b.release(n.tolist())
    paged.paged_release(table, n, free, fc, 16)
    _same(b, table, free, fc, "released")


def test_most_requests(dev):
    # 65,535 requests: the running sums span many chunks
    import tabicl_mi355_paged as paged
    N, R = 65535, 16
    count = (torch.arange(N, device=dev) % 3).to(I32)
    n = torch.full((N,), 15, dtype=I32, device=dev)
    table = torch.full((N, 2), -1, dtype=I32, device=dev)
    table[:, 0] = torch.arange(N, device=dev)
    P = 2 * N
    free = torch.arange(P, device=dev).to(I32)
    free[:N] = torch.arange(N, P, device=dev).to(I32)
    fc = torch.tensor([N], dtype=I32, device=dev)
    granted = paged.paged_reserve(table, n, count, free, fc, R)
    assert torch.equal(granted, count)
    need = count > 1
    rank = need.long().cumsum(0) - 1
    assert torch.equal(table[:, 1].long(), torch.where(need, P - 1 - rank, -1)) and int(fc) == N - int(need.sum())
    total = int(count.sum())
    slots, starts = paged.paged_slots(table, n, count, total, P, R)
    ends = count.long().cumsum(0)
    assert torch.equal(starts[1:].long(), ends) and int(starts[0]) == 0
    seq = torch.searchsorted(ends, torch.arange(total, device=dev), right=True)
    row = 15 + torch.arange(total, device=dev) - starts.long()[seq]
    assert torch.equal(slots, table.long()[seq, row // R] * R + row % R)


def test_slots_of_a_smaller_total(dev):
    # fewer places than rows: those that there are
    import tabicl_mi355_paged as paged
    table, n, free, fc, g = _books(dev, 5, [0, 40, 3], 6, 16, spare=9)
    count = torch.tensor([30, 2, 50], dtype=I32, device=dev)
    _step(table, n, count, free, fc, 16, total=31, what="smaller")
    slots, starts = paged.paged_slots(table, n, count, 0, free.numel(), 16)
    assert slots.shape == (0,) and starts.tolist() == [0, 30, 32, 82]
    slots, starts = paged.paged_slots(table[:0], n[:0], count[:0], 4, free.numel(), 16)
    assert slots.tolist() == [-1] * 4 and starts.tolist() == [0]
    wide = torch.full((3, 9), 1, dtype=I32, device=dev)
    wide[:, :6] = table
    assert paged.paged_slots(wide[:, :6], n, count, 82, free.numel(), 16)[0].tolist() == paged.paged_slots(table, n, count, 82, free.numel(), 16)[0].tolist()


@pytest.mark.parametrize("code", [BF, F32, E4, I8], ids=["bf16", "fp32", "e4m3", "int8"])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_append_packed(dev, code, D):
    import tabicl_mi355_paged as paged
    H, R = 3, 16
    table, n, free, fc, _ = _books(dev, D, [0, 20, 5, 33], 8, R, spare=3)
    g = torch.Generator(device=dev).manual_seed(D)
    count = torch.tensor([18, 0, 40, 7], dtype=I32, device=dev)
    paged.paged_reserve(table, n, count, free, fc, R)  # too few pages: some rows have no place
    P, total = free.numel(), 65 + 4
    slots, starts = paged.paged_slots(table, n, count, total, P, R)
    assert (slots[:65] == -1).any() and (slots[65:] == -1).all()
    q8 = code in (E4, I8)
    kp, vp = ((torch.randn(P, H, R, D, generator=g, device=dev) * 20).to(code) for _ in range(2))
    scales = torch.full((P, H, 2), 2.0 ** -6, device=dev) if q8 else None
    dtype = BF if q8 else code
    kv = torch.randn(total, 2, H, D, generator=g, device=dev).to(dtype)
    for k, v in ((kv[:, 0], kv[:, 1]), (kv[:, 1].contiguous(), kv[:, 0].expand(total, H, D))):
        before = kp.clone(), vp.clone()
        if q8:
            want = ref.append(kp.cpu(), vp.cpu(), scales.cpu(), table.cpu(), n.cpu(), k.cpu(), v.cpu(), count.cpu(), starts.cpu())
        paged.paged_append_packed(kp, vp, table, n, count, k, v, slots, starts, scales)
        torch.cuda.synchronize()
        if q8:
            assert torch.equal(kp.float().double().cpu(), want[0]) and torch.equal(vp.float().double().cpu(), want[1])
            assert torch.equal(scales.cpu(), want[2])
            continue
        for pages, x, old in ((kp, k, before[0]), (vp, v, before[1])):
            for j, s in enumerate(slots.tolist()):
                if s >= 0:
                    old[s // R, :, s % R] = x[j]
            assert torch.equal(pages, old)


def test_append_slots_out_of_range(dev):
    import tabicl_mi355_paged as paged
    kp, vp = (torch.zeros(3, 2, 16, 64, dtype=BF, device=dev) for _ in range(2))
    k = torch.ones(4, 2, 64, dtype=BF, device=dev)
    slots = torch.tensor([-1, 47, 48, 2 ** 62], dtype=torch.int64, device=dev)
    z = torch.zeros(1, dtype=I32, device=dev)
    paged.paged_append_packed(kp, vp, z.view(1, 1), z, z, k, k, slots, torch.zeros(2, dtype=I32, device=dev))
    torch.cuda.synchronize()
    for t in (kp, vp):
        assert (t[2, :, 15] == 1).all() and int(t.sum()) == 128


@pytest.mark.parametrize("code", [BF, E4], ids=["bf16", "e4m3"])
def test_captured_service(dev, code):
    # one graph: pages for the rows, the rows into them, bounds, attention over all pages and over chosen ones, and requests that
    # are done give their pages back; replayed with other rows while the requests grow, against the books in Python
    import tabicl_mi355_paged as paged
    N, H, R, D, M, total = 4, 2, 16, 64, 8, 40
    P = 20
    q8 = code is E4
    g = torch.Generator(device=dev).manual_seed(1)
    table = torch.full((N, M), -1, dtype=I32, device=dev)
    free = torch.arange(P, dtype=I32, device=dev)
    fc = torch.tensor([P], dtype=I32, device=dev)
    n, count, keep = (torch.zeros(N, dtype=I32, device=dev) for _ in range(3))
    kp, vp = (torch.zeros(P, H, R, D, device=dev).to(code) for _ in range(2))
    scales = torch.zeros(P, H, 2, device=dev) if q8 else None
    bnd, bs = torch.zeros(P, H, 2, D, dtype=torch.int8, device=dev), torch.zeros(P, H, device=dev)
    k, v = (torch.zeros(total, H, D, dtype=BF, device=dev) for _ in range(2))
    q = torch.zeros(N, H, 1, D, dtype=BF, device=dev)

    def step():
        granted = paged.paged_reserve(table, n, count, free, fc, R)
        slots, starts = paged.paged_slots(table, n, count, total, P, R)
        paged.paged_append_packed(kp, vp, table, n, count, k, v, slots, starts, scales)
        grown = n + granted
        paged.paged_bounds(kp, table, grown, bnd, bs, n, total, scales)
        out = paged.paged_attention(q, kp, vp, table, grown, scales=scales)
        index = paged.paged_select(q, bnd, bs, table, grown, R, 2)
        few = paged.paged_sparse_attention(q, kp, vp, table, grown, index, scales=scales)
        n.copy_(torch.minimum(grown, keep))
        paged.paged_release(table, n, free, fc, R)
        return granted, slots, starts, out, index, few, grown

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    b = ref.Books(table.tolist(), free.tolist(), int(fc), P, R)
    wk, wv = kp.cpu(), vp.cpu()
    ws = scales.cpu() if q8 else None
    lengths = n.tolist()
    plans = [([10, 0, 20, 3], [99] * 4), ([1, 1, 1, 1], [99, 99, 0, 99]), ([7, 30, 2, 1], [99] * 4), ([0, 0, 0, 40], [99] * 4),
             ([20, 5, 5, 5], [9, 99, 99, 99]), ([12, 13, 14, 1], [99] * 4), ([1, 1, 1, 1], [0, 0, 0, 5])]
    for i, (new, stay) in enumerate(plans):
        count.copy_(torch.tensor(new, dtype=I32))
        keep.copy_(torch.tensor(stay, dtype=I32))
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=g, device=dev).to(BF))
        graph.replay()
        torch.cuda.synchronize()
        granted, slots, starts, out, index, few, grown = got
        assert granted.tolist() == b.reserve(lengths, new), i
        s, st = b.slots(lengths, new, total)
        assert slots.tolist() == s and starts.tolist() == st, i
        t = torch.tensor(b.table, dtype=I32)
        if q8:
            wk, wv, ws = (x.to(code) if j < 2 else x for j, x in
                          enumerate(ref.append(wk, wv, ws, t, lengths, k.cpu(), v.cpu(), new, st)))
        else:
            for pages, x in ((wk, k.cpu()), (wv, v.cpu())):
                for j, slot in enumerate(s):
                    if slot >= 0:
                        pages[slot // R, :, slot % R] = x[j]
        assert torch.equal(kp.cpu().view(torch.uint8), wk.view(torch.uint8)), i
        assert torch.equal(vp.cpu().view(torch.uint8), wv.view(torch.uint8)), i
        lengths = [a + x for a, x in zip(lengths, granted.tolist())]
        assert grown.tolist() == lengths
        kk, vv = (ref.values(w, ws, j) if q8 else w.double() for j, w in enumerate((wk, wv)))
        want, _, tol, _ = paged_ref.attention(q.cpu(), kk, vv, t, lengths, D ** -0.5)
        paged_ref.near(out, want, tol, f"step {i}")
        assert torch.equal(index.cpu(), ref.select(q, bnd, bs, t, lengths, R, 2)), i
        want, tol = ref.sparse_attention(q.cpu(), kk, vv, t, lengths, index.cpu(), D ** -0.5)
        paged_ref.near(few, want, tol, f"step {i}, two pages")
        lengths = [min(a, x) for a, x in zip(lengths, stay)]
        b.release(lengths)
        _same(b, table, free, fc, i)
        assert n.tolist() == lengths


def test_ops_equal_direct_calls_and_compile(dev):
    import tabicl_mi355_paged as paged
    from torch.utils._python_dispatch import TorchDispatchMode

    class Seen(TorchDispatchMode):
        names: list = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.names.append(str(func))
            return func(*args, **(kwargs or {}))

    def make():
        table, n, free, fc, _ = _books(dev, 9, [5, 30, 0], 6, 16, spare=20)
        g = torch.Generator(device=dev).manual_seed(2)
        kp, vp = (torch.zeros(free.numel(), 2, 16, 64, dtype=BF, device=dev) for _ in range(2))
        k = torch.randn(50, 2, 64, generator=g, device=dev).to(BF)
        return table, n, free, fc, torch.tensor([20, 3, 27], dtype=I32, device=dev), kp, vp, k

    def step(table, n, free, fc, count, kp, vp, k):
        granted = paged.paged_reserve(table, n, count, free, fc, 16)
        slots, starts = paged.paged_slots(table, n, count, 50, kp.shape[0], 16)
        paged.paged_append_packed(kp, vp, table, n, count, k, k, slots, starts)
        paged.paged_release(table, n + 9, free, fc, 16)
        return granted, slots, starts

    def ops(*a):
        with Seen():
            return step(*a)

    results = []
    for f in (step, ops, torch.compile(step, fullgraph=True)):
        a = make()
        r = f(*a)
        torch.cuda.synchronize()
        results.append([t.clone() for t in (*r, *a)])
    for other in results[1:]:
        for x, y in zip(results[0], other):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    for name in ("paged_reserve", "paged_slots", "paged_append_slots", "paged_release"):
        assert any(name in s for s in Seen.names), (name, Seen.names)


def test_native_calls_equal_python_ones(dev, monkeypatch):
    # the calls that the native module makes against the same ones without it
    import tabicl_mi355_native as nat
    import tabicl_mi355_paged as paged
    nat.load()
    assert nat.DIRECT is not None, "tabicl_mi355_direct.so is built beside the library"

    def step(code):
        table, n, free, fc, _ = _books(dev, 3, [50, 300, 0, 17], 40, 16, spare=90)
        P, H, D, R = free.numel(), 2, 64, 16
        g = torch.Generator(device=dev).manual_seed(5)
        kp, vp = (torch.zeros(P, H, R, D, device=dev).to(code) for _ in range(2))
        scales = torch.ones(P, H, 2, device=dev) if code in (E4, I8) else None
        count = torch.tensor([20, 100, 33, 1], dtype=I32, device=dev)
        out = [paged.paged_reserve(table, n, count, free, fc, R), *paged.paged_slots(table, n, count, 160, P, R)]
        x = torch.randn(160, H, D, generator=g, device=dev).to(BF if scales is not None else code)
        paged.paged_append_packed(kp, vp, table, n, count, x, -x, *out[1:], scales)
        n = n + count
        bnd, bs = torch.zeros(P, H, 2, D, dtype=torch.int8, device=dev), torch.zeros(P, H, device=dev)
        paged.paged_bounds(kp, table, n, bnd, bs, None, None, scales)
        q = torch.randn(4, 2 * H, 3, D, generator=g, device=dev).to(BF if code in (E4, I8) else code)
        out.append(paged.paged_select(q, bnd, bs, table, n, R, 5))
        out.append(paged.paged_sparse_attention(q, kp, vp, table, n, out[-1], scales=scales))
        if scales is not None:
            more = torch.randn(4, H, 2, D, generator=g, device=dev)
            paged.paged_append(kp, vp, table, n - 1, more, more * 9, scales=scales)
            out.append(paged.paged_attention(q, kp, vp, table, n, scales=scales))
            live = torch.arange(333, device=dev).view(1, 1, -1, 1) < n.view(-1, 1, 1, 1)  # nothing is written past a length
            out.extend(torch.where(live, x, 0.0) for x in paged.paged_gather(kp, vp, table, n, 333, scales=scales, dtype=F32))
        paged.paged_release(table, n - 30, free, fc, R)
        torch.cuda.synchronize()
        return [t for t in (*out, table, free, fc, kp, vp, scales, bnd, bs) if t is not None]

    for code in (BF, F32, E4, I8):
        with_it = step(code)
        with monkeypatch.context() as m:
            m.setattr(nat, "DIRECT", None)
            without = step(code)
        for a, b in zip(with_it, without):
            assert a.dtype == b.dtype and torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8)), code


def test_two_graphs(dev):
    # two captured services replayed in turn and together: nothing is shared between them
    import tabicl_mi355_paged as paged
    runs = []
    for seed in (1, 2):
        table, n, free, fc, _ = _books(dev, seed, [40, 200, 0], 30, 16, spare=60)
        P = free.numel()
        g = torch.Generator(device=dev).manual_seed(seed)
        kp, vp = (torch.randn(P, 8, 16, 64, generator=g, device=dev).to(E4) for _ in range(2))
        scales = torch.ones(P, 8, 2, device=dev)
        q = torch.randn(3, 8, 1, 64, generator=g, device=dev).to(BF)
        count = torch.tensor([3, 1, 9], dtype=I32, device=dev)
        bnd, bs = torch.zeros(P, 8, 2, 64, dtype=torch.int8, device=dev), torch.zeros(P, 8, device=dev)

        def step(table=table, n=n, free=free, fc=fc, kp=kp, vp=vp, scales=scales, q=q, count=count, bnd=bnd, bs=bs):
            granted = paged.paged_reserve(table, n, count, free, fc, 16)
            paged.paged_bounds(kp, table, n, bnd, bs, None, None, scales)
            index = paged.paged_select(q, bnd, bs, table, n, 16, 4)
            outs = granted, index, paged.paged_sparse_attention(q, kp, vp, table, n, index, scales=scales), \
                paged.paged_attention(q, kp, vp, table, n, scales=scales)
            paged.paged_release(table, n, free, fc, 16)
            return outs

        want = [t.clone() for t in step()]
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = step()
        runs.append((graph, got, want, stream))
    torch.cuda.synchronize()
    for together in (False, True, True):
        for graph, got, _, stream in runs:
            for t in got:
                t.view(torch.uint8).fill_(7)
        torch.cuda.synchronize()
        for graph, _, _, stream in runs:
            with torch.cuda.stream(stream if together else torch.cuda.current_stream()):
                graph.replay()
        torch.cuda.synchronize()
        for _, got, want, _ in runs:
            for a, b in zip(got, want):
                assert torch.equal(a, b)
