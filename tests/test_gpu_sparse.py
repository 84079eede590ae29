"""GPU tests of attention over selected pages against the plain forms of paged8_ref.py: bounds of the pages' keys, the pages of
largest bound, attention over listed pages, and the three together.

Bounds and selections are whole numbers and compared exactly. Attention is held to paged_ref.attention's bound over the rows
of the listed pages."""
import math

import pytest
import torch

import paged8_ref as ref
import paged_ref
from test_gpu_paged8 import BF, E4, F32, I8, _pool

pytestmark = pytest.mark.gpu
FORMATS = pytest.mark.parametrize("fmt", [BF, F32, E4, I8], ids=["bf16", "fp32", "e4m3", "int8"])


def _case(dev, seed, lengths, H=4, G=1, D=64, R=32, T=1, fmt=BF, dtype=None, slack=0, spare=4):
    """Pages in random order; everything that no sequence holds is NaN (codes: 127)."""
    g = torch.Generator(device=dev).manual_seed(seed)
    N, M = len(lengths), max(1, max(-(-n // R) for n in lengths)) + slack
    P = N * M + spare
    table = torch.randperm(P, generator=g, device=dev)[:N * M].to(torch.int32).view(N, M).contiguous()
    scales = None
    if fmt in (E4, I8):
        kp, vp = (_pool(dev, g, P, H, R, D, fmt) for _ in range(2))
        scales = torch.exp2(torch.randint(-9, -4, (P, H, 2), generator=g, device=dev).float())
    else:
        kp, vp = ((torch.randn(P, H, R, D, generator=g, device=dev) + torch.randn(P, H, 1, D, generator=g, device=dev)).to(fmt)
                  for _ in range(2))
    dead = torch.ones(P, R, dtype=torch.bool, device=dev)
    for n, length in enumerate(lengths):
        _, page, row = paged_ref.rows_of(table[n], length, R, P)
        dead[page, row] = False
    for t in (kp, vp):
        if scales is None:
            t.masked_fill_(dead[:, None, :, None], math.nan)
        else:
            t.view(torch.uint8).masked_fill_(dead[:, None, :, None], 127)
    dtype = dtype or (fmt if scales is None else BF)
    q = (torch.randn(N, H * G, T, D, generator=g, device=dev) * 1.5).to(dtype)
    return q, kp, vp, scales, table, torch.tensor(lengths, dtype=torch.int32, device=dev), g


def _values(kp, scales, which):
    return kp.double() if scales is None else ref.values(kp, scales, which)


def _fresh(kp, g):
    P, H, _, D = kp.shape
    return (torch.randint(-127, 128, (P, H, 2, D), generator=g, device=kp.device, dtype=torch.int8),
            torch.rand(P, H, generator=g, device=kp.device))


def _check_bounds(kp, scales, table, n, bnd, bs, before, start=None):
    want = ref.bounds(_values(kp, scales, 0).cpu(), table.cpu(), n.cpu(), None if start is None else start.cpu())
    b, s = bnd.cpu(), bs.cpu()
    wb, ws = before[0].cpu().clone(), before[1].cpu().clone()
    for (page, h), (hi, lo, step) in want.items():
        wb[page, h, 0], wb[page, h, 1], ws[page, h] = hi.to(torch.int8), lo.to(torch.int8), step
    assert torch.equal(s, ws)
    assert torch.equal(b, wb)


EDGES = [0, 1, 15, 16, 17, 31, 32, 33, 64, 100, 255, 256, 257]


@FORMATS
@pytest.mark.parametrize("D,R", [(32, 16), (64, 32), (64, 256), (128, 64), (128, 16)])
def test_bounds(dev, fmt, D, R):
    import tabicl_mi355_paged as paged
    q, kp, vp, scales, table, n, g = _case(dev, D + R, EDGES, D=D, R=R, fmt=fmt, slack=1)
    bnd, bs = _fresh(kp, g)
    before = bnd.clone(), bs.clone()
    paged.paged_bounds(kp, table, n, bnd, bs, scales=scales)
    _check_bounds(kp, scales, table, n, bnd, bs, before)


def test_bounds_of_part(dev):
    # pages before `start` keep theirs; start past the end, below 0; a bound on the rows
    import tabicl_mi355_paged as paged
    q, kp, vp, scales, table, n, g = _case(dev, 3, [300, 90, 64, 10, 33], R=16, slack=1)
    bnd, bs = _fresh(kp, g)
    before = bnd.clone(), bs.clone()
    start = torch.tensor([290, 80, 64, -5, 2 ** 31 - 1], dtype=torch.int32, device=dev)
    paged.paged_bounds(kp, table, n, bnd, bs, start, 10)
    _check_bounds(kp, scales, table, n, bnd, bs, before, start)
    before = bnd.clone(), bs.clone()
    paged.paged_bounds(kp, table, n, bnd, bs, start)
    _check_bounds(kp, scales, table, n, bnd, bs, before, start)


def test_bounds_special(dev):
    # infinite and NaN keys, zero pages, the ends of the scales, pages outside the pool
    import tabicl_mi355_paged as paged
    q, kp, vp, scales, table, n, g = _case(dev, 5, [200, 200, 50], R=16, fmt=F32)
    kp[table[0, 0].long(), 0, 3, 5] = math.inf
    kp[table[0, 0].long(), 0, 4, 6] = -math.inf
    kp[table[0, 1].long(), 1, :, 7] = math.nan
    kp[table[0, 2].long(), 2, 0] = math.nan
    kp[table[0, 3].long(), 0] = 0.0
    kp[table[0, 4].long(), 1] *= 1e-25
    kp[table[0, 5].long(), 2] *= 1e35
    kp[table[0, 6].long(), 3] = math.nan
    kp[table[0, 7].long(), 3] = math.inf
    table[1, 4], table[1, 5], table[2, 0] = -1, kp.shape[0], -2 ** 31
    bnd, bs = _fresh(kp, g)
    before = bnd.clone(), bs.clone()
    paged.paged_bounds(kp, table, n, bnd, bs)
    _check_bounds(kp, scales, table, n, bnd, bs, before)


def _check_select(q, bnd, bs, table, n, R, K, what=""):
    import tabicl_mi355_paged as paged
    print(f"[sparse] select {what} q {tuple(q.shape)} pages {tuple(bnd.shape)} table {tuple(table.shape)} K {K}", flush=True)
    got = paged.paged_select(q, bnd, bs, table, n, R, K)
    torch.cuda.synchronize()
    want = ref.select(q, bnd, bs, table.cpu(), n.cpu(), R, K)
    assert got.dtype == torch.int32 and torch.equal(got.cpu(), want), what
    return got


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("T,G", [(1, 1), (2, 1), (7, 1), (16, 1), (33, 1), (1, 4), (5, 3), (2, 8), (1, 16), (2, 17), (1, 40)])
def test_select(dev, dtype, D, T, G):
    q, kp, vp, scales, table, n, g = _case(dev, D + T, [700, 0, 33, 1], H=2, G=G, D=D, R=16, T=T, dtype=dtype, slack=1)
    bnd, bs = _fresh(kp, g)
    bs = torch.exp2(torch.randint(-3, 2, bs.shape, generator=g, device=dev).float())
    for K in (1, 3, 43, 44, 50):
        _check_select(q, bnd, bs, table, n, 16, K, f"T {T} G {G}")


@pytest.mark.parametrize("pages,T", [(900, 3), (3000, 9), (9000, 2), (20000, 4), (32768, 1), (33000, 2)])
def test_select_of_many_pages(dev, pages, T):
    # tables for which fewer query rows' codes fit in LDS, and one whose codes do not fit at all
    g = torch.Generator(device=dev).manual_seed(pages)
    P, H, D, R = pages + 7, 1, 32, 16
    table = torch.randperm(P, generator=g, device=dev)[:2 * (pages // 2)].to(torch.int32).view(1, -1)
    table = torch.cat((table, table.flip(1)), 0)
    n = torch.tensor([table.shape[1] * R - 5, table.shape[1] * R // 3], dtype=torch.int32, device=dev)
    bnd = torch.randint(-20, 21, (P, H, 2, D), generator=g, device=dev, dtype=torch.int8)
    bs = torch.ones(P, H, device=dev)
    q = torch.randn(2, H, T, D, generator=g, device=dev).to(BF)
    for K in (1, 64, 1000):
        _check_select(q, bnd, bs, table, n, R, K, "many")


def test_select_ties_and_special(dev):
    # all bounds equal; bounds that differ in the sign of 0; NaN, infinite and zero queries; pages outside the pool
    q, kp, vp, scales, table, n, g = _case(dev, 9, [500, 400, 300], H=2, R=16, T=4, slack=2)
    bnd, bs = torch.ones_like(_fresh(kp, g)[0]), torch.ones(kp.shape[0], 2, device=dev)
    _check_select(q, bnd, bs, table, n, 16, 7, "equal")
    bnd = torch.randint(-1, 2, bnd.shape, generator=g, device=dev, dtype=torch.int8)
    q[0, :, 0], q[0, :, 1, 3], q[1, 0, 2, :5], q[2, 1, 3] = 0, math.nan, math.inf, math.nan
    q[2, 0, 1, 7] = -math.inf
    table[0, 3:9], table[1, 5], table[2, :18] = -1, kp.shape[0], 2 ** 31 - 1
    n[1] = 2 ** 31 - 1
    for K in (1, 5, 11, 30, 40):
        _check_select(q, bnd, bs, table, n, 16, K, "special")
    _check_select(q * 1e-20, bnd, bs, table, n, 16, 6, "small")
    _check_select(q.float() * 1e30, bnd, bs * 2.0 ** 100, table, n, 16, 6, "great")


def _check_sparse(q, kp, vp, scales, table, n, index, scale=None, what=""):
    import tabicl_mi355_paged as paged
    print(f"[sparse] attention {what} q {tuple(q.shape)} pool {tuple(kp.shape)} {q.dtype} {kp.dtype} index {tuple(index.shape)}",
          flush=True)
    out = paged.paged_sparse_attention(q, kp, vp, table, n, index, scale, scales=scales)
    torch.cuda.synchronize()
    want, tol = ref.sparse_attention(q, _values(kp, scales, 0), _values(vp, scales, 1), table, n, index,
                                     q.shape[-1] ** -0.5 if scale is None else scale)
    paged_ref.near(out, want, tol, what)
    return out


@FORMATS
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("T,G,R,K", [(1, 1, 16, 1), (1, 1, 64, 9), (3, 4, 32, 5), (2, 17, 16, 40), (5, 1, 256, 3)])
def test_attention(dev, fmt, D, T, G, R, K):
    # random lists: any order, pages twice, none, outside the table, past the length
    q, kp, vp, scales, table, n, g = _case(dev, D + T + R, [900, 0, 5, 300], H=2, G=G, D=D, R=R, T=T, fmt=fmt, slack=1)
    M = table.shape[1]
    index = torch.randint(-1, M + 1, (4, 2, T, K), generator=g, device=dev, dtype=torch.int32)
    index[0, 0, 0] = -1
    index[3, 1, T - 1, 0] = 2 ** 31 - 1
    table[3, 2 % M] = -1
    out = _check_sparse(q, kp, vp, scales, table, n, index, what="lists")
    assert (out[1] == 0).all() and (out[0, :G, 0] == 0).all()
    if scales is not None:
        _check_sparse(q.float(), kp, vp, scales, table, n, index, 0.2, what="fp32 queries")


@FORMATS
@pytest.mark.parametrize("lengths,T,K", [([20000], 1, 100), ([5000, 300, 9000], 2, 33), ([3000] * 40, 4, 8)])
def test_select_and_attend(dev, fmt, lengths, T, K):
    import tabicl_mi355_paged as paged
    q, kp, vp, scales, table, n, g = _case(dev, T, lengths, H=8, T=T, R=64, fmt=fmt)
    bnd, bs = _fresh(kp, g)
    before = bnd.clone(), bs.clone()
    paged.paged_bounds(kp, table, n, bnd, bs, scales=scales)
    _check_bounds(kp, scales, table, n, bnd, bs, before)
    index = _check_select(q, bnd, bs, table, n, 64, K)
    _check_sparse(q, kp, vp, scales, table, n, index, what="selected")
    every = paged.paged_select(q, bnd, bs, table, n, 64, table.shape[1])  # all pages: attention over the whole cache
    out = paged.paged_sparse_attention(q, kp, vp, table, n, every, scales=scales)
    want, _, tol, _ = paged_ref.attention(q, _values(kp, scales, 0), _values(vp, scales, 1), table, n, 64 ** -0.5)
    paged_ref.near(out, want, tol, "every page")


def test_bound_holds(dev):
    # no key of a page scores above its bound, but for the rounding of the query to its step: the heaviest page is chosen
    import tabicl_mi355_paged as paged
    q, kp, vp, scales, table, n, g = _case(dev, 17, [4000, 4000], H=4, T=3, R=32)
    kp[table[:, 77].long(), :, 5] = (q[:, :, 0] * 9).to(BF)  # a key that answers query row 0
    bnd, bs = _fresh(kp, g)
    paged.paged_bounds(kp, table, n, bnd, bs)
    index = paged.paged_select(q, bnd, bs, table, n, 32, 2)
    assert (index[:, :, 0] == 77).any(-1).all()
    out = paged.paged_sparse_attention(q, kp, vp, table, n, index)
    dense = paged.paged_attention(q, kp, vp, table, n)
    assert (out[:, :, 0].float() - dense[:, :, 0].float()).abs().max() <= 2.0 ** -6 * dense[:, :, 0].float().abs().max()


def test_strided_outputs_and_streams(dev):
    import tabicl_mi355_paged as paged
    q, kp, vp, scales, table, n, g = _case(dev, 21, [900, 65, 300], T=5)
    bnd, bs = _fresh(kp, g)
    paged.paged_bounds(kp, table, n, bnd, bs)
    index = paged.paged_select(q, bnd, bs, table, n, 32, 4)
    want = paged.paged_sparse_attention(q, kp, vp, table, n, index)
    N, H, T, D = q.shape
    odd = torch.zeros(q.numel() + 1, dtype=BF, device=dev)[1:].view(q.shape).copy_(q)
    proj = torch.zeros(N, T, H, D, dtype=BF, device=dev).copy_(q.transpose(1, 2)).transpose(1, 2)
    for x in (odd, proj):
        assert torch.equal(paged.paged_select(x, bnd, bs, table, n, 32, 4), index)
        assert torch.equal(paged.paged_sparse_attention(x, kp, vp, table, n, index), want)
    out = torch.empty(N, T, H, D, dtype=BF, device=dev).transpose(1, 2)
    assert paged.paged_sparse_attention(q, kp, vp, table, n, index, out=out) is out and torch.equal(out, want)
    over = q.clone()
    paged.paged_sparse_attention(over, kp, vp, table, n, index, out=over)
    assert torch.equal(over, want)
    wide = torch.full((N, table.shape[1] + 3), -1, dtype=torch.int32, device=dev)
    wide[:, :table.shape[1]] = table
    view = wide[:, :table.shape[1]]  # rows of a wider table
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        i2 = paged.paged_select(q, bnd, bs, view, n, 32, 4)
        got = paged.paged_sparse_attention(q, kp, vp, view, n, i2)
    torch.cuda.synchronize()
    assert torch.equal(i2, index) and torch.equal(got, want)


def test_large_offsets(dev):
    import tabicl_mi355_paged as paged
    P, H, R, D = 2200, 8, 4096, 64
    kp, vp = (torch.empty(P, H, R, D, dtype=E4, device=dev) for _ in range(2))
    scales = torch.ones(P, H, 2, device=dev)
    ids = torch.tensor([[2199, 0], [2100, 2198]], dtype=torch.int32, device=dev)
    g = torch.Generator(device=dev).manual_seed(1)
    for p in ids.flatten().tolist():
        kp[p], vp[p] = (_pool(dev, g, 1, H, R, D, E4)[0] for _ in range(2))
    n = torch.tensor([8000, 5000], dtype=torch.int32, device=dev)
    q = torch.randn(2, H, 2, D, generator=g, device=dev).to(BF) * 2.0 ** -7
    bnd, bs = torch.zeros(P, H, 2, D, dtype=torch.int8, device=dev), torch.zeros(P, H, device=dev)
    paged.paged_bounds(kp, ids, n, bnd, bs, scales=scales)
    small = torch.arange(4, dtype=torch.int32, device=dev).view(2, 2)
    four = ids.flatten().long()
    want = ref.bounds(torch.cat([kp[p:p + 1].float() for p in four.tolist()]).double().cpu(), small.cpu(), n.cpu())
    for (i, h), (hi, lo, step) in want.items():
        assert torch.equal(bnd[four[i], h].double().cpu(), torch.stack((hi, lo))) and float(bs[four[i], h]) == step
    index = paged.paged_select(q, bnd, bs, ids, n, R, 1)
    out = paged.paged_sparse_attention(q, kp, vp, ids, n, index, scales=scales)
    sub = [torch.cat([t.view(torch.uint8)[p:p + 1] for p in four.tolist()]).view(E4) for t in (kp, vp)]
    w, tol = ref.sparse_attention(q, sub[0].float().double(), sub[1].float().double(), small, n, index, D ** -0.5)
    paged_ref.near(out, w, tol, "far pages")


def test_graph_and_ops(dev):
    import tabicl_mi355_paged as paged
    from torch.utils._python_dispatch import TorchDispatchMode
    q, kp, vp, scales, table, n, g = _case(dev, 71, [3000, 900, 20], H=8, T=2, slack=2)
    kp.nan_to_num_(nan=0.5)
    vp.nan_to_num_(nan=0.5)
    bnd, bs = _fresh(kp, g)
    start = [bnd.clone(), bs.clone()]
    view = torch.empty(3, 2, 8, 64, dtype=BF, device=dev).transpose(1, 2)

    def step():
        paged.paged_bounds(kp, table, n, bnd, bs, (n - 40).clamp(min=0), 50)
        index = paged.paged_select(q, bnd, bs, table, n, 32, 6)
        paged.paged_sparse_attention(q, kp, vp, table, n, index, 0.3, view)
        return index, paged.paged_sparse_attention(q, kp, vp, table, n, index), view

    def reset():
        bnd.copy_(start[0])
        bs.copy_(start[1])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()

    class Seen(TorchDispatchMode):
        names: list = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.names.append(str(func))
            return func(*args, **(kwargs or {}))

    def ops():
        with Seen():
            return step()

    for i in range(3):
        q.copy_(torch.randn(q.shape, generator=g, device=dev).to(BF))
        n.copy_(torch.tensor([3000 - 700 * i, 900 + i, 20 * i], dtype=torch.int32))
        table.copy_(table.flip(0) if i == 1 else table)
        results = []
        for run in (lambda: (graph.replay(), got)[1], step, ops):
            reset()
            torch.cuda.synchronize()
            r = run()
            torch.cuda.synchronize()
            results.append([t.clone() for t in (*r, bnd, bs)])
        for other in results[1:]:
            for x, y in zip(results[0], other):
                assert torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8)), f"replay {i}"
    for name in ("paged_bounds", "paged_select", "paged_sparse_attn.", "paged_sparse_attn_out"):
        assert any(name in s for s in Seen.names), (name, Seen.names)


def test_compile(dev):
    import tabicl_mi355_paged as paged
    q, kp, vp, scales, table, n, g = _case(dev, 77, [300, 20], fmt=E4)
    bnd, bs = _fresh(kp, g)

    def step(q, kp, vp, scales, table, n, bnd, bs):
        paged.paged_bounds(kp, table, n, bnd, bs, scales=scales)
        index = paged.paged_select(q, bnd, bs, table, n, 32, 3)
        out = torch.zeros_like(q)
        paged.paged_sparse_attention(q * 2, kp, vp, table, n, index, None, out, scales)
        return out + 1, index, paged.paged_sparse_attention(q, kp, vp, table, n, index, scales=scales)

    start = bnd.clone(), bs.clone()
    want = [t.clone() for t in (*step(q, kp, vp, scales, table, n, bnd, bs), bnd, bs)]
    bnd.copy_(start[0])
    bs.copy_(start[1])
    got = (*torch.compile(step, fullgraph=True)(q, kp, vp, scales, table, n, bnd, bs), bnd, bs)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def test_nothing_to_do(dev):
    import tabicl_mi355_paged as paged
    q, kp, vp, scales, table, n, g = _case(dev, 79, [40, 5], H=2, R=16, T=2)
    bnd, bs = _fresh(kp, g)
    assert paged.paged_select(q, bnd, bs, table, n, 16, 0).shape == (2, 2, 2, 0)
    assert (paged.paged_sparse_attention(q, kp, vp, table, n, torch.empty(2, 2, 2, 0, dtype=torch.int32, device=dev)) == 0).all()
    assert paged.paged_select(q[:, :, :0], bnd, bs, table, n, 16, 3).shape == (2, 2, 0, 3)
    assert paged.paged_select(q[:0], bnd, bs, table[:0], n[:0], 16, 3).shape == (0, 2, 2, 3)
    for b, s, t in ((bnd, bs, table[:, :0]), (bnd[:0], bs[:0], table)):
        index = paged.paged_select(q, b, s, t, n, 16, 3)
        assert (index == -1).all()
    paged.paged_bounds(kp, table[:, :0], n, bnd, bs)
    paged.paged_bounds(kp[:0], table, n, bnd[:0], bs[:0])
    assert (paged.paged_sparse_attention(q, kp[:0], vp[:0], table, n, index) == 0).all()
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [BF, I8], ids=["bf16", "int8"])
def test_cache_selects(dev, dtype):
    # PagedIclKVCache(select=K): queries are those of the functions over its own pages, in a graph too
    import tabicl_mi355_paged as paged
    g = torch.Generator(device=dev).manual_seed(6)
    S, H, D, R, K = 3, 8, 64, 16, 4
    c = paged.PagedIclKVCache(S, 2, H, D, 600, 90, R, dtype, dev, select=K)
    for new in ([20, 10, 0], [1, 1, 1], [300, 40, 70]):
        for b in range(2):
            k, v = (torch.randn(S, H, max(new), D, generator=g, device=dev).to(BF) for _ in range(2))
            if new[0] == 300:
                pick = [torch.cat([x[s, :, :new[s]].transpose(0, 1) for s in range(S)]) for x in (k, v)]
                c.append_packed(b, *pick, new)
            else:
                c.append(b, k, v, new)
    scales = None if c.scales is None else c.scales[1]
    want = ref.bounds(_values(c.keys[1], scales, 0).cpu(), c.table.cpu(), c.lengths[1].cpu())
    for (page, h), (hi, lo, step) in want.items():
        assert torch.equal(c.bounds[1][page, h].double().cpu(), torch.stack((hi, lo))) and float(c.bound_scales[1][page, h]) == step
    q = torch.randn(S, H, 3, D, generator=g, device=dev).to(BF)
    out = c.query(1, q)
    index = ref.select(q, c.bounds[1], c.bound_scales[1], c.table.cpu(), c.lengths[1].cpu(), R, K).to(dev)
    o, tol = ref.sparse_attention(q, _values(c.keys[1], scales, 0), _values(c.values[1], scales, 1), c.table, c.lengths[1], index,
                                  D ** -0.5)
    paged_ref.near(out, o, tol, "cache")
    few = c.query(1, q, K * R)  # no more rows than the selection holds: all of them
    assert (few.float() - out.float()).abs().max() > 0
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = c.query(1, q)
    graph.replay()
    torch.cuda.synchronize()
    paged_ref.near(got, o, tol, "captured")
    for b in range(2):
        c.append(b, k[:, :, :5], v[:, :, :5])
    graph.replay()  # the cache has grown
    torch.cuda.synchronize()
    index = ref.select(q, c.bounds[1], c.bound_scales[1], c.table.cpu(), c.lengths[1].cpu(), R, K).to(dev)
    o, tol = ref.sparse_attention(q, _values(c.keys[1], scales, 0), _values(c.values[1], scales, 1), c.table, c.lengths[1], index,
                                  D ** -0.5)
    paged_ref.near(got, o, tol, "captured, grown")


@FORMATS
@pytest.mark.parametrize("N,H,T,G,D,R,K", [(90, 8, 1, 1, 64, 16, 9), (5, 2, 60, 3, 64, 32, 20), (40, 8, 2, 1, 128, 64, 9),
                                           (3, 1, 400, 1, 32, 16, 1), (2, 2, 1, 1, 128, 64, 5)])
def test_many_items(dev, fmt, N, H, T, G, D, R, K):
    # items in number and length as the waves of a workgroup are chosen by; lists longer and shorter than a sequence's pages
    g = torch.Generator().manual_seed(N)
    lengths = torch.randint(0, 700, (N,), generator=g).tolist()
    q, kp, vp, scales, table, n, g = _case(dev, N + T, lengths, H=H, G=G, D=D, R=R, T=T, fmt=fmt)
    bnd, bs = _fresh(kp, g)
    index = _check_select(q, bnd, bs, table, n, R, K, "many items")
    _check_sparse(q, kp, vp, scales, table, n, index, what="many items")


@pytest.mark.parametrize("pages,K", [(33000, 33000), (40, 5000), (2000, 2000)])
def test_select_every_page(dev, pages, K):
    # no more pages than are asked for: all of them, whatever their bounds; some are not there
    g = torch.Generator(device=dev).manual_seed(pages)
    P, R = pages + 7, 16
    table = torch.randperm(P, generator=g, device=dev)[:pages].to(torch.int32).view(1, -1).repeat(2, 1)
    table[:, 3:20] = -1
    table[1, pages - 1] = P
    n = torch.tensor([pages * R, pages * R - 40], dtype=torch.int32, device=dev)
    bnd = torch.randint(-20, 21, (P, 1, 2, 32), generator=g, device=dev, dtype=torch.int8)
    bs = torch.ones(P, 1, device=dev)
    bs[::3] = math.nan
    q = torch.randn(2, 1, 3, 32, generator=g, device=dev).to(BF)
    import tabicl_mi355_paged as paged
    got = paged.paged_select(q, bnd, bs, table, n, R, K).cpu()
    for i, count in enumerate((pages, pages - 2)):
        ids = table[i, :count].cpu()
        there = torch.nonzero((ids >= 0) & (ids < P)).view(-1).int()
        want = torch.full((K,), -1, dtype=torch.int32)
        want[:len(there)] = there
        assert (got[i] == want).all()


@pytest.mark.parametrize("pages", [32768, 15000])
def test_select_of_many_wide_pages(dev, pages):
    # the most LDS that a workgroup takes: all codes of the longest table beside the queries and bounds of 128 dims
    g = torch.Generator(device=dev).manual_seed(pages)
    table = torch.randperm(pages, generator=g, device=dev).to(torch.int32).view(1, -1)
    n = torch.tensor([pages * 16 - 3], dtype=torch.int32, device=dev)
    bnd = torch.randint(-20, 21, (pages, 1, 2, 128), generator=g, device=dev, dtype=torch.int8)
    q = torch.randn(1, 2, 2, 128, generator=g, device=dev).to(BF)
    _check_select(q, bnd, torch.ones(pages, 1, device=dev), table, n, 16, 100, "many wide pages")
