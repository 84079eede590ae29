"""GPU tests of the 8-bit paged K/V cache against the plain forms of paged8_ref.py: attention over e4m3 and int8 codes at the
tiles' and pages' edges, rows written into pages that are new, partly full or of a smaller scale, and read back, with
non-finite values, strided and packed rows, in captured graphs, far into a large pool.

Codes and scales are compared exactly. Attention is held to paged_ref.attention's bound over the values that the codes stand
for: products of codes are exact, fp32 queries and probabilities enter as three bf16 terms that lose nothing, and the bf16
ones as the two terms that the bound counts."""
import pytest
import torch

import paged8_ref as ref
import paged_ref

pytestmark = pytest.mark.gpu
BF, F32, E4, I8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn, torch.int8
CODES = pytest.mark.parametrize("code", [E4, I8], ids=["e4m3", "int8"])
DTYPES = pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])


def _pool(dev, g, P, H, R, D, code):
    x = torch.randn(P, H, R, D, generator=g, device=dev)
    return (x * 100).clamp(-448, 448).to(E4) if code is E4 else (x * 30).round().clamp(-127, 127).to(I8)


def _case(dev, seed, lengths, H=8, G=1, D=64, R=64, T=1, dtype=BF, code=E4, spare=5, slack=0, sharp=1.0):
    """A pool whose pages lie in random order; the codes of rows that nobody holds are NaN (int8: as large as can be), and so
    are the scales of pages that nobody holds."""
    g = torch.Generator(device=dev).manual_seed(seed)
    N = len(lengths)
    M = max(1, max(-(-n // R) for n in lengths)) + slack
    P = N * M + spare
    table = torch.randperm(P, generator=g, device=dev)[:N * M].to(torch.int32).view(N, M).contiguous()
    kp, vp = (_pool(dev, g, P, H, R, D, code) for _ in range(2))
    scales = torch.exp2(torch.randint(-10, -3, (P, H, 2), generator=g, device=dev).float())
    dead = torch.ones(P, R, dtype=torch.bool, device=dev)
    for n, length in enumerate(lengths):
        _, page, row = paged_ref.rows_of(table[n], length, R, P)
        dead[page, row] = False
    for t in (kp, vp):
        t.view(torch.uint8).masked_fill_(dead[:, None, :, None], 127)
    scales.masked_fill_(dead.all(1)[:, None, None], float("nan"))
    q = (torch.randn(N, H * G, T, D, generator=g, device=dev) * sharp).to(dtype)
    return q, kp, vp, scales, table, torch.tensor(lengths, dtype=torch.int32, device=dev), g


def _attend(q, kp, vp, scales, table, lengths, scale=None, what=""):
    import tabicl_mi355_paged as paged
    keep = [t.clone() for t in (q, kp, vp, scales, table, lengths)]
    print(f"[paged8] {what} q {tuple(q.shape)} pool {tuple(kp.shape)} {q.dtype} {kp.dtype}", flush=True)
    out = paged.paged_attention(q, kp, vp, table, lengths, None, scale, scales=scales)
    torch.cuda.synchronize()
    assert out.shape == q.shape and out.dtype == q.dtype
    for t, k in zip((q, kp, vp, scales, table, lengths), keep):
        assert torch.equal(t.contiguous().view(torch.uint8), k.contiguous().view(torch.uint8))
    want, _, tol, _ = paged_ref.attention(q, ref.values(kp, scales, 0), ref.values(vp, scales, 1), table, lengths,
                                          q.shape[-1] ** -0.5 if scale is None else scale)
    paged_ref.near(out, want, tol, what)
    return out


EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 512, 513, 1000, 1023, 1025]


@DTYPES
@CODES
@pytest.mark.parametrize("R", [16, 64, 256])
def test_lengths(dev, dtype, code, R):
    out = _attend(*_case(dev, R, EDGES, H=2, R=R, dtype=dtype, code=code, sharp=2.0)[:-1], what="lengths")
    assert (out[0] == 0).all()
    short = [n for n in EDGES if n <= 700]
    _attend(*_case(dev, R + 1, short, H=2, R=R, dtype=dtype, code=code, sharp=2.0)[:-1], what="short")


@DTYPES
@CODES
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("T,G", [(1, 1), (1, 4), (5, 3), (16, 1), (17, 1), (33, 2), (65, 1)])
def test_query_rows_and_head_dims(dev, dtype, code, D, T, G):
    _attend(*_case(dev, 7 * D + T, [300, 77, 1], H=3, G=G, D=D, R=32, T=T, dtype=dtype, code=code, sharp=1.5)[:-1], what="short")
    _attend(*_case(dev, 7 * D + T, [1300, 77, 0], H=3, G=G, D=D, R=32, T=T, dtype=dtype, code=code, sharp=1.5)[:-1], what="split")


@DTYPES
@CODES
@pytest.mark.parametrize("lengths,T", [([45001], 1), ([20011, 3, 9999, 0, 12345], 2), ([6007] * 3, 40)])
def test_long_and_ragged(dev, dtype, code, lengths, T):
    _attend(*_case(dev, T, lengths, R=64, T=T, dtype=dtype, code=code, slack=3, sharp=2.5)[:-1], what="long")


@CODES
def test_many_pages_per_workgroup(dev, code):
    # pages of 16 rows by the thousand: the 64 page ids and scales at a time are loaded anew on the way
    _attend(*_case(dev, 3, [70001, 40000], H=1, R=16, T=3, code=code, sharp=2.0)[:-1], what="small pages")


@CODES
def test_pages_without_rows(dev, code):
    q, kp, vp, scales, table, n, g = _case(dev, 11, [200, 150, 90, 64], H=2, R=16, code=code, T=2)
    table[0, 3], table[0, 7], table[1, :] = -1, kp.shape[0], -5
    table[2, 0], table[2, 6:] = 2 ** 31 - 1, -1
    n[3] = -7
    out = _attend(q, kp, vp, scales, table, n, what="holes")
    assert (out[1] == 0).all() and (out[3] == 0).all()
    q, kp, vp, scales, table, n, g = _case(dev, 12, [48, 48], H=2, R=16, code=code)
    want = _attend(q, kp, vp, scales, table, n, what="full")
    n[:] = torch.tensor([2 ** 31 - 1, 49], dtype=torch.int32)  # clamped to the table
    assert torch.equal(_attend(q, kp, vp, scales, table, n, what="past the table"), want)


@DTYPES
def test_strided_views_and_outputs(dev, dtype):
    import tabicl_mi355_paged as paged
    N, H, T, D = 3, 4, 5, 64
    q, kp, vp, scales, table, n, g = _case(dev, 21, [100, 65, 2000], H=H, T=T, R=32, dtype=dtype)
    want = _attend(q, kp, vp, scales, table, n, what="contiguous")
    proj = torch.zeros(N, T, 3 * H * D, dtype=dtype, device=dev)
    proj[:, :, :H * D] = q.transpose(1, 2).reshape(N, T, H * D)
    odd = torch.zeros(N * H * T * D + 1, dtype=dtype, device=dev)[1:].view(N, H, T, D).copy_(q)
    for x in (proj[:, :, :H * D].view(N, T, H, D).transpose(1, 2), odd):
        assert torch.equal(paged.paged_attention(x, kp, vp, table, n, scales=scales), want)
    out = torch.full((N, T, H, D), 7.0, dtype=dtype, device=dev).transpose(1, 2)
    assert paged.paged_attention(q, kp, vp, table, n, out=out, scales=scales) is out and torch.equal(out, want)
    over = q.clone()
    paged.paged_attention(over, kp, vp, table, n, out=over, scales=scales)
    assert torch.equal(over, want)
    # pages of several blocks behind each other, one taken out of the middle
    big = torch.zeros(kp.shape[0], 3, *kp.shape[1:], dtype=torch.uint8, device=dev)
    big[:, 1] = kp.view(torch.uint8)
    bigv = torch.zeros_like(big)
    bigv[:, 1] = vp.view(torch.uint8)
    assert torch.equal(paged.paged_attention(q, big[:, 1].view(kp.dtype), bigv[:, 1].view(kp.dtype), table, n, scales=scales), want)


def test_non_finite(dev):
    # a NaN code makes the rows of its head NaN, and those alone; infinite queries
    import tabicl_mi355_paged as paged
    q, kp, vp, scales, table, n, g = _case(dev, 31, [100, 2000], H=2, T=2)
    kp.view(torch.uint8)[table[0, 0].long(), 1, 3, 5] = 127
    vp.view(torch.uint8)[table[1, 2].long(), 0, 1, 9] = 255
    out = paged.paged_attention(q, kp, vp, table, n, scales=scales)
    assert torch.isnan(out[0, 1]).all() and torch.isfinite(out[0, 0]).all()
    assert torch.isnan(out[1, 0, :, 9]).all() and torch.isfinite(out[1, 0, :, :9]).all() and torch.isfinite(out[1, 1]).all()


@DTYPES
@CODES
@pytest.mark.parametrize("scale", [0.5, 0.0, -0.125, 3.0])
def test_scale_of_the_scores(dev, dtype, code, scale):
    _attend(*_case(dev, 41, [700, 33, 3000], H=2, T=3, dtype=dtype, code=code)[:-1], scale=scale, what="scale")


@CODES
def test_scales_of_any_size(dev, code):
    # the ends of their range, other than powers of two, and one page of great values among small ones
    q, kp, vp, scales, table, n, g = _case(dev, 43, [500, 90], H=2, T=2, R=16, code=code)
    scales[..., 0] = 2.0 ** -9
    for s in (2.0 ** -60, 2.0 ** 60, 2.0 ** 100):
        scales[..., 1] = s
        _attend(q, kp, vp, scales, table, n, what=f"V scale {s}")
    scales[..., 1] = torch.rand(scales.shape[:2], generator=g, device=dev) * 0.01 + 1e-3
    scales[table[0, 4].long()] = 0.07
    _attend(q, kp, vp, scales, table, n, what="mixed")
    scales[table[0, 7].long(), :, 1] = 1e30
    _attend(q, kp, vp, scales, table, n, what="one great page")


def test_repeatable_and_concurrent(dev):
    import tabicl_mi355_paged as paged
    a = _case(dev, 51, [9000, 300], T=4)[:-1]
    b = _case(dev, 52, [20, 7000], T=4, code=I8, dtype=F32)[:-1]
    call = lambda c: paged.paged_attention(c[0], c[1], c[2], c[4], c[5], scales=c[3])  # noqa: E731
    want = call(a), call(b)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = [None, None]
        for i, (s, c) in enumerate(zip(streams, (a, b))):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got[i] = call(c)
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# ---------------------------------------------------------------------------------------------
# rows in and out
# ---------------------------------------------------------------------------------------------
def _same_pools(kp, vp, scales, want, what):
    wk, wv, ws = want
    bad = [x for x, a, b in (("k", kp.float().double(), wk), ("v", vp.float().double(), wv), ("scales", scales, ws))
           if not torch.equal(torch.nan_to_num(a, nan=1e9).cpu(), torch.nan_to_num(b, nan=1e9).cpu())]
    assert not bad, f"{what}: {bad}"


def _append(kp, vp, scales, table, n, k, v, count=None, what=""):
    import tabicl_mi355_paged as paged
    want = ref.append(kp.cpu(), vp.cpu(), scales.cpu(), table.cpu(), n.cpu(), k.cpu(), v.cpu(), None if count is None else count.cpu())
    print(f"[paged8] append {what} {tuple(k.shape)} pool {tuple(kp.shape)} {k.dtype} {kp.dtype}", flush=True)
    paged.paged_append(kp, vp, table, n, k, v, count, scales=scales)
    torch.cuda.synchronize()
    _same_pools(kp, vp, scales, want, what)


@DTYPES
@CODES
@pytest.mark.parametrize("D,R", [(32, 16), (64, 64), (128, 32), (64, 256), (128, 256)])
@pytest.mark.parametrize("starts,T", [([0, 0], 1), ([5, 63], 1), ([16, 300], 70), ([0, 31], 300), ([255, 1], 2)])
def test_append(dev, dtype, code, D, R, starts, T):
    # rows of growing size, so that pages that hold rows are rounded again; NaN wherever nobody wrote
    g = torch.Generator(device=dev).manual_seed(T + D)
    H = 2
    M = -(-(max(starts) + T) // R)
    P = 2 * M + 3
    kp, vp = (_pool(dev, g, P, H, R, D, code) for _ in range(2))
    scales = torch.exp2(torch.randint(-10, -3, (P, H, 2), generator=g, device=dev).float())
    table = torch.randperm(P, generator=g, device=dev)[:2 * M].to(torch.int32).view(2, M)
    n = torch.tensor(starts, dtype=torch.int32, device=dev)
    for i, size in enumerate((0.2, 30.0, 1e-4)):
        k, v = ((torch.randn(2, H, T, D, generator=g, device=dev) * size * torch.rand(2, H, 1, 1, generator=g, device=dev)).to(dtype)
                for _ in range(2))
        count = None if i != 1 else torch.tensor([T - 1, T], dtype=torch.int32, device=dev)
        _append(kp, vp, scales, table, n, k, v, count, what=f"pass {i}")


@CODES
def test_append_row_by_row(dev, code):
    # pages filled one row at a time are rounded again whenever a larger row comes: at most half a step each time, with steps
    # that double, so all in all less than one step of the final scale
    import tabicl_mi355_paged as paged
    g = torch.Generator(device=dev).manual_seed(9)
    H, R, D, L = 2, 32, 64, 50
    kp, vp = (torch.zeros(4, H, R, D, dtype=code, device=dev) for _ in range(2))
    scales = torch.zeros(4, H, 2, device=dev)
    table = torch.tensor([[2, 0]], dtype=torch.int32, device=dev)
    k, v = (torch.randn(1, H, L, D, generator=g, device=dev) * torch.exp2(torch.arange(L, device=dev) / 7.0)[:, None] for _ in range(2))
    for t in range(L):
        n = torch.tensor([t], dtype=torch.int32, device=dev)
        _append(kp, vp, scales, table, n, k[:, :, t:t + 1], v[:, :, t:t + 1], what=f"row {t}")
    n = torch.tensor([L], dtype=torch.int32, device=dev)
    got = paged.paged_gather(kp, vp, table, n, L, scales=scales, dtype=F32)
    for which, (a, b) in enumerate(zip(got, (k, v))):
        step = scales[table[0].long(), :, which].repeat_interleave(R, 0)[:L].t()[None, :, :, None]  # [1, H, L, 1]
        if code is I8:
            assert ((a - b).abs() <= step).all()
        else:  # half a step of four significant bits, and the subnormals' steps: 2^-9 of the scale in all
            assert ((a - b).abs() <= b.abs() * 2.0 ** -4 + step * 2.0 ** -9).all()


@CODES
def test_append_special_values(dev, code):
    g = torch.Generator(device=dev).manual_seed(10)
    kp, vp = (_pool(dev, g, 3, 2, 16, 32, code) for _ in range(2))
    scales = torch.ones(3, 2, 2, device=dev)
    table = torch.tensor([[1, 2]], dtype=torch.int32, device=dev)
    n = torch.tensor([0], dtype=torch.int32, device=dev)
    for size in (0.0, 1e-30, 3e-18, 2.0 ** -66, 1.0, 448.0, 449.0, 127.0, 127.5, 1e20, 1e33, 3e38):
        k, v = (torch.randn(1, 2, 20, 32, generator=g, device=dev).clamp(-0.99, 0.99) * size for _ in range(2))
        k[0, 0, 3, 4], k[0, 1, 2, 1], v[0, 0, 17, 3] = size, -size, size
        _append(kp, vp, scales, table, n, k, v, what=f"size {size}")
        k[0, 0, 1, 1], k[0, 0, 2, 2], k[0, 0, 2, 3], v[0, 1] = float("nan"), float("inf"), float("-inf"), float("nan")
        _append(kp, vp, scales, table, n, k, v, what=f"size {size} with NaN")
    # values half way between two codes
    half = (torch.arange(-64, 64, device=dev).float() + 0.5).view(1, 2, 2, 32)
    half[..., 0] = 127.0
    _append(kp, vp, scales, table, n, half, half, what="half steps")


@CODES
def test_append_layouts_and_holes(dev, code):
    g = torch.Generator(device=dev).manual_seed(12)
    N, H, T, D, R = 3, 2, 40, 64, 16
    kp, vp = (_pool(dev, g, 12, H, R, D, code) for _ in range(2))
    scales = torch.ones(12, H, 2, device=dev) * 2.0 ** -8
    table = torch.tensor([[1, 2, 3], [4, -1, 5], [6, 12, 7]], dtype=torch.int32, device=dev)
    n = torch.tensor([5, 15, -3], dtype=torch.int32, device=dev)
    count = torch.tensor([99, 20, -1], dtype=torch.int32, device=dev)  # more than T, more than fits, less than none
    kv = torch.randn(N, T, 2, H, D, generator=g, device=dev).to(BF)
    k, v = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
    _append(kp, vp, scales, table, n, k, v, count, what="heads of a projection")
    _append(kp, vp, scales, table, n, k, v, None, what="all rows")
    odd = torch.zeros(N * H * T * D + 1, dtype=BF, device=dev)[1:].view(N, H, T, D).copy_(k)
    one = torch.randn(N, H, 1, D, generator=g, device=dev).to(BF).expand(N, H, T, D)
    _append(kp, vp, scales, table, n, odd, one, count, what="odd")
    last = torch.tensor([48, 1000, 2 ** 31 - 1], dtype=torch.int32, device=dev)  # no room
    _append(kp, vp, scales, table, last, k, v, None, what="full")


@DTYPES
@CODES
@pytest.mark.parametrize("D,R,L", [(32, 16, 70), (64, 64, 200), (128, 32, 65)])
def test_gather(dev, dtype, code, D, R, L):
    import tabicl_mi355_paged as paged
    q, kp, vp, scales, table, n, g = _case(dev, 61, [L, 0, 33], H=3, D=D, R=R, code=code)
    table[2, 1 if R < 33 else 0] = -1
    if code is E4:
        kp.view(torch.uint8)[table[0, 0].long(), 0, 2, 3] = 255
    for rows in (0, 1, L, L + 9):
        k, v = paged.paged_gather(kp, vp, table, n, rows, scales=scales, dtype=dtype)
        assert k.dtype == dtype and k.shape == (3, 3, rows, D)
        for which, (pages, got) in enumerate(((kp, k), (vp, v))):
            x = ref.values(pages, scales, which)
            for s in range(3):
                at, page, row = paged_ref.rows_of(table[s], min(int(n[s]), rows), R, kp.shape[0])
                want = torch.zeros(min(int(n[s]), rows), 3, D, dtype=torch.float64, device=dev)
                want[at] = x[page, :, row]
                assert torch.equal(torch.nan_to_num(got[s, :, :len(want)].double(), nan=1e9),
                                   torch.nan_to_num(want.transpose(0, 1), nan=1e9))


def test_large_offsets(dev):
    # pages more than 2^32 codes apart in one pool
    import tabicl_mi355_paged as paged
    P, H, R, D = 2200, 8, 4096, 64
    kp, vp = (torch.empty(P, H, R, D, dtype=E4, device=dev) for _ in range(2))
    scales = torch.ones(P, H, 2, device=dev)
    ids = torch.tensor([[2199, 0], [2100, 2198]], dtype=torch.int32, device=dev)
    g = torch.Generator(device=dev).manual_seed(1)
    k, v = (torch.randn(2, H, 5000, D, generator=g, device=dev).to(BF) for _ in range(2))
    zero, n = (torch.tensor(x, dtype=torch.int32, device=dev) for x in ([0, 0], [5000, 5000]))
    paged.paged_append(kp, vp, ids, zero, k, v, scales=scales)
    gk, gv = paged.paged_gather(kp, vp, ids, n, 5000, scales=scales, dtype=F32)
    for s in range(2):
        for which, (x, got) in enumerate(((k, gk), (v, gv))):
            for p in range(2):
                lo, hi = p * R, min(5000, (p + 1) * R)
                most = x[s, :, lo:hi].float().abs().amax((1, 2)).tolist()
                step = torch.tensor([2.0 ** ref.exponent(m, 448.0) for m in most], dtype=torch.float64, device=dev)
                assert torch.equal(scales[ids[s, p].long(), :, which].double(), step)
                want = ref.codes(x[s, :, lo:hi].double() / step[:, None, None], E4) * step[:, None, None]
                assert torch.equal(got[s, :, lo:hi].double(), want)
    q = torch.randn(2, H, 2, D, generator=g, device=dev).to(BF)
    out = paged.paged_attention(q, kp, vp, ids, n, scales=scales)
    for s in range(2):
        one, length = torch.zeros(1, 1, dtype=torch.int32, device=dev), torch.tensor([5000])
        want, _, tol, _ = paged_ref.attention(q[s:s + 1], gk[s:s + 1], gv[s:s + 1], one, length, D ** -0.5)
        paged_ref.near(out[s:s + 1], want, tol, "far pages")


def test_graph_and_ops(dev):
    # append, attention and gather in one graph, replayed with other rows, lengths and pages; the ops give the same
    import tabicl_mi355_paged as paged
    from torch.utils._python_dispatch import TorchDispatchMode
    q, kp, vp, scales, table, n, g = _case(dev, 71, [3000, 900, 20], T=2, slack=2)
    scales.nan_to_num_(nan=1.0)
    k, v = (torch.randn(3, 8, 10, 64, generator=g, device=dev).to(BF) for _ in range(2))
    grown = n + 10
    start = [t.clone() for t in (kp, vp, scales)]
    view = torch.empty(3, 2, 8, 64, dtype=BF, device=dev).transpose(1, 2)

    def step():
        paged.paged_append(kp, vp, table, n, k, v, scales=scales)
        out = paged.paged_attention(q, kp, vp, table, grown, scales=scales)
        paged.paged_attention(q, kp, vp, table, grown, None, 0.3, view, scales)
        rows = paged.paged_gather(kp, vp, table, grown.clamp(max=16), 16, scales=scales)
        return (out, view, rows[0][:, :, :10], rows[1][:, :, :10])

    def reset():
        for t, s in zip((kp, vp, scales), start):
            t.copy_(s)

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
        k.copy_(torch.randn(k.shape, generator=g, device=dev).to(BF) * 10.0 ** i)
        n.copy_(torch.tensor([3000 - 700 * i, 900 + i, 20 * i], dtype=torch.int32))
        grown.copy_(n + 10)
        table.copy_(table.flip(0) if i == 1 else table)
        results = []
        for run in (lambda: (graph.replay(), got)[1], step, ops):
            reset()
            torch.cuda.synchronize()
            r = run()
            torch.cuda.synchronize()
            results.append([t.clone() for t in (*r, kp, vp, scales)])
        for other in results[1:]:
            for x, y in zip(results[0], other):
                assert torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8)), f"replay {i}"
    for name in ("paged_append_q8", "paged_attn_q8.", "paged_attn_q8_out", "paged_gather_q8"):
        assert any(name in s for s in Seen.names), (name, Seen.names)


def test_compile(dev):
    import tabicl_mi355_paged as paged
    q, kp, vp, scales, table, n, g = _case(dev, 77, [300, 20], code=I8)
    scales.nan_to_num_(nan=1.0)
    start = [t.clone() for t in (kp, vp, scales)]

    def step(q, kp, vp, scales, table, n):
        paged.paged_append(kp, vp, table, n - 2, q, q, scales=scales)
        out = torch.zeros_like(q)
        paged.paged_attention(q * 2, kp, vp, table, n, None, None, out, scales)
        return out + 1, paged.paged_attention(q, kp, vp, table, n, scales=scales)

    want = [t.clone() for t in (*step(q, kp, vp, scales, table, n), kp, vp, scales)]
    for t, s in zip((kp, vp, scales), start):
        t.copy_(s)
    got = (*torch.compile(step, fullgraph=True)(q, kp, vp, scales, table, n), kp, vp, scales)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_nothing_to_do(dev):
    import tabicl_mi355_paged as paged
    q, kp, vp, scales, table, n, g = _case(dev, 79, [40, 5], H=2, R=16, T=2)
    assert paged.paged_attention(q[:0], kp, vp, table[:0], n[:0], scales=scales).shape == (0, 2, 2, 64)
    assert paged.paged_attention(q[:, :, :0], kp, vp, table, n, scales=scales).shape == (2, 2, 0, 64)
    for pool, s, t in (((kp, vp), scales, table[:, :0]), ((kp[:0], vp[:0]), scales[:0], table)):
        assert (paged.paged_attention(q, *pool, t, n, scales=s) == 0).all()
        paged.paged_append(*pool, t, n, q, q, scales=s)
        assert paged.paged_gather(*pool, t, n, 0, scales=s)[0].shape == (2, 2, 0, 64)
    torch.cuda.synchronize()


# ---------------------------------------------------------------------------------------------
# PagedIclKVCache
# ---------------------------------------------------------------------------------------------
@CODES
def test_cache_together(dev, code):
    # appends (padded, counted, packed), queries of few and of many rows, a release, a query in a graph
    import tabicl_mi355_paged as paged
    g = torch.Generator(device=dev).manual_seed(4)
    S, B, H, D, R = 3, 2, 8, 64, 32
    c = paged.PagedIclKVCache(S, B, H, D, 900, 90, R, code, dev)
    rows = [[] for _ in range(S)]
    for i, new in enumerate(([300, 10, 0], [1, 1, 1], [200, 70, 31])):
        for b in range(B):
            ks = [torch.randn(r, H, D, generator=g, device=dev).to(BF) for r in new]
            vs = [torch.randn(r, H, D, generator=g, device=dev).to(BF) for r in new]
            if i == 1:
                c.append(b, torch.stack(ks).transpose(1, 2), torch.stack(vs).transpose(1, 2))
            elif i == 0:
                pad = lambda xs: torch.nn.utils.rnn.pad_sequence(xs, batch_first=True).transpose(1, 2)  # noqa: E731
                c.append(b, pad(ks), pad(vs), new)
            else:
                c.append_packed(b, torch.cat(ks), torch.cat(vs), new)
            if b == 1:
                for s in range(S):
                    rows[s].append((ks[s], vs[s]))
    assert [c.length(1, s) for s in range(S)] == [501, 81, 32]

    def check(q, out, seqs=range(S)):
        for s in seqs:
            k, v = (torch.cat([r[j] for r in rows[s]]).double() for j in range(2))
            p = torch.softmax(torch.matmul(q[s].double(), k.permute(1, 2, 0)) * D ** -0.5, -1)
            want = torch.matmul(p, v.transpose(0, 1))
            # e4m3 rounds each key and value by up to 2^-4 of itself, int8 by half of 1/64 of a page's largest: errors that
            # average over 64 dims and 30 rows and more; the bound is a tenth of the values' size
            assert float((out[s].double() - want).abs().mean()) < 0.1
            assert float((out[s].double() - want).abs().max()) < 1.0

    for T, dtype in ((1, BF), (3, F32), (1100, BF)):
        q = torch.randn(S, H, T, D, generator=g, device=dev).to(dtype)
        out = c.query(1, q)
        assert out.dtype == dtype
        check(q, out)
        k, v = paged.paged_gather(*c.block_kv(1), c.table, c.lengths[1], 501, scales=c.scales[1], dtype=F32)
        want, _, tol, _ = paged_ref.attention(q, k, v, torch.arange(S, dtype=torch.int32, device=dev).view(S, 1), c.lengths[1], D ** -0.5)
        if T < 1000:
            paged_ref.near(out, want, tol, f"cache T {T}")
        else:  # the dense kernel takes bf16 probabilities: 2^-8 of each value
            most = max(float(v[s, :, :c.length(1, s)].abs().max()) for s in range(S))  # nothing is written past a length
            assert ((out.double() - want).abs() <= tol + 2.0 ** -8 * most).all()
    q = torch.randn(S, H, 2, D, generator=g, device=dev).to(BF)
    want = c.query(1, q)
    # of fewer rows a sequence's keys are shared among other waves: the same terms summed in another order, each sum within the
    # tolerance of the exact value, so within twice of it of each other
    k, v = paged.paged_gather(*c.block_kv(1), c.table, c.lengths[1], 501, scales=c.scales[1], dtype=F32)
    _, _, tol, _ = paged_ref.attention(q, k, v, torch.arange(S, dtype=torch.int32, device=dev).view(S, 1), c.lengths[1], D ** -0.5)
    assert ((c.estimators(1, 3).query(1, q[1:]).double() - want[1:].double()).abs() <= 2 * tol[1:]).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = c.query(1, q)
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert (got.double() - want.double()).abs().max() < 2.0 ** -6  # another split of the work
    free = c.free_pages
    c.release(0)
    assert c.free_pages > free and (c.query(1, q)[0] == 0).all()


def test_cache_layers(dev):
    # attention_layer and query_blocks over a cache in 8 bits are those of a bf16 cache that holds the same values
    import tabicl_mi355_icl as icl
    import tabicl_mi355_paged as paged
    g = torch.Generator(device=dev).manual_seed(5)
    S, H, D, W = 2, 8, 64, 512
    c8 = paged.PagedIclKVCache(S, 1, H, D, 300, 24, 32, I8, dev)
    c16 = paged.PagedIclKVCache(S, 1, H, D, 300, 24, 32, BF, dev)
    rnd = lambda *s: torch.randn(*s, generator=g, device=dev) * 0.05  # noqa: E731
    w = icl.IclBlockWeights(torch.ones(W, device=dev), torch.zeros(W, device=dev), rnd(3 * W, W).to(BF), rnd(3 * W).to(BF),
                            rnd(W, W).to(BF), rnd(W).to(BF), torch.ones(W, device=dev), torch.zeros(W, device=dev),
                            rnd(2 * W, W).to(BF), rnd(2 * W).to(BF), rnd(W, 2 * W).to(BF), rnd(W).to(BF))
    x = torch.randn(S, 250, W, generator=g, device=dev).to(BF)
    c8.append_projected(0, x, w.in_w, w.in_b)
    k, v = paged.paged_gather(*c8.block_kv(0), c8.table, c8.lengths[0], 250, scales=c8.scales[0])
    c16.append(0, k, v)
    t = torch.randn(S, 3, W, generator=g, device=dev)
    a, b = c8.query_blocks(t, [w]), c16.query_blocks(t, [w])
    assert a.dtype == b.dtype and float((a - b).abs().max()) <= 2.0 ** -6 * float(b.abs().max())
    a, b = (c.attention_layer(0, t.to(BF), w.in_w, w.in_b, w.out_w, w.out_b) for c in (c8, c16))
    assert a.dtype == BF and float((a - b).abs().max()) <= 2.0 ** -6 * float(b.abs().max())


@CODES
@pytest.mark.parametrize("N,most,H,T,D,dtype", [
    (600, 20, 1, 1, 64, BF), (600, 250, 1, 3, 32, F32), (40, 200, 8, 40, 64, BF), (40, 130, 8, 40, 128, BF),  # two waves an item
    (3, 500, 2, 5, 64, BF), (70, 700, 8, 2, 64, F32), (40, 600, 8, 33, 32, BF), (20, 1000, 8, 70, 128, BF),    # four
    (2, 1000, 8, 1, 128, F32), (1, 777, 2, 200, 64, BF),                                                       # eight
    (3, 1500, 2, 70, 128, BF), (3, 1500, 2, 70, 128, F32), (2, 2100, 2, 33, 64, F32), (2, 1300, 2, 100, 32, F32),  # split, wide tiles
])
def test_items_and_tiles(dev, code, N, most, H, T, D, dtype):
    # sequences in number and length as the variants are chosen by: waves of an item, query rows of a tile
    g = torch.Generator().manual_seed(N + most)
    lengths = torch.randint(0, most + 1, (N,), generator=g).tolist()
    lengths[0] = most
    _attend(*_case(dev, most, lengths, H=H, T=T, D=D, R=16, dtype=dtype, code=code, sharp=2.0)[:-1], what="items")


@CODES
@pytest.mark.parametrize("R,D", [(128, 128), (256, 128), (512, 64), (512, 128), (1024, 128)])
def test_append_to_large_pages(dev, code, R, D):
    # as many values of a page as 256 or 512 threads keep, and more; non-finite ones among them, rows held before
    g = torch.Generator(device=dev).manual_seed(R + D)
    H, T = 2, 2 * R + 3
    kp, vp = (_pool(dev, g, 9, H, R, D, code) for _ in range(2))
    scales = torch.exp2(torch.randint(-10, -3, (9, H, 2), generator=g, device=dev).float())
    table = torch.tensor([[7, 0, 3, 5], [1, 8, 2, 6]], dtype=torch.int32, device=dev)
    n = torch.tensor([R - 5, 0], dtype=torch.int32, device=dev)
    k, v = (torch.randn(2, H, T, D, generator=g, device=dev) * 3.0 for _ in range(2))
    k[0, 0, 2], k[1, 1, R + 1, 3], v[0, 1, R // 2, 5], v[1, 0, T - 1] = float("inf"), float("nan"), -float("inf"), float("nan")
    for dtype in (F32, BF):
        _append(kp, vp, scales, table, n, k.to(dtype), v.to(dtype), what=f"large pages {dtype}")
