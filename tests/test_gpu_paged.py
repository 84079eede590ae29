"""GPU tests of the paged K/V cache (tabicl_mi355_paged) against the plain float64 forms of paged_ref.py: attention of
few rows with and without the weights it adds up, append and eviction, at lengths around the tiles' and pages' edges, on
strided inputs, with pages that hold no rows, with non-finite values in and around the live rows, on other streams, in
captured graphs, far into a large pool, and run together as PagedIclKVCache runs them.

Everything the kernels must not read (rows past a length, pages nobody holds) is NaN; everything they must not write is
compared. Bounds: paged_ref.attention derives them; append and eviction copy, so they are compared bit for bit."""
import pytest
import torch

import paged_ref as ref

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _case(dev, seed, lengths, H=8, G=1, D=64, R=64, T=1, dtype=BF, spare=5, slack=0, blocks=None, sharp=1.0):
    """A pool whose pages lie in random order, NaN wherever no sequence has a row."""
    g = torch.Generator(device=dev).manual_seed(seed)
    N = len(lengths)
    M = max(1, max(-(-n // R) for n in lengths)) + slack
    P = N * M + spare
    table = torch.randperm(P, generator=g, device=dev)[:N * M].to(torch.int32).view(N, M).contiguous()
    lead = () if blocks is None else (blocks,)
    kp, vp = (torch.randn(*lead, P, H, R, D, generator=g, device=dev).to(dtype) for _ in range(2))
    dead = torch.ones(P, R, dtype=torch.bool, device=dev)
    for n, length in enumerate(lengths):
        _, page, row = ref.rows_of(table[n], length, R, P)
        dead[page, row] = False
    for t in (kp, vp):
        t.masked_fill_(dead[:, None, :, None], float("nan"))
    q = (torch.randn(N, H * G, T, D, generator=g, device=dev) * sharp).to(dtype)
    return q, kp, vp, table, torch.tensor(lengths, dtype=torch.int32, device=dev), g


def _attend(q, kp, vp, table, lengths, weights=None, scale=None, what=""):
    import tabicl_mi355_paged as paged
    before = None if weights is None else weights.clone()
    keep = [t.clone() for t in (q, kp, vp, table, lengths)]
    print(f"[paged] {what} q {tuple(q.shape)} pool {tuple(kp.shape)} {q.dtype}", flush=True)
    out = paged.paged_attention(q, kp, vp, table, lengths, weights, scale)
    torch.cuda.synchronize()
    assert out.shape == q.shape and out.dtype == q.dtype
    for t, k in zip((q, kp, vp, table, lengths), keep):
        assert torch.equal(t.view(torch.uint8) if t.is_contiguous() else t, k.view(torch.uint8) if t.is_contiguous() else k)
    want, w, tol, wtol = ref.attention(q, kp, vp, table, lengths, q.shape[-1] ** -0.5 if scale is None else scale, before)
    ref.near(out, want, tol, what + " out")
    if weights is not None:
        ref.near(weights, w, wtol, what + " weights")
        for n in range(len(lengths)):  # past the length: left alone
            assert torch.equal(weights[n, max(0, int(lengths[n])):], before[n, max(0, int(lengths[n])):])
    return out


EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 512, 513, 1000, 1023, 1025]


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("R", [16, 64, 256])
@pytest.mark.parametrize("weighted", [False, True], ids=["", "weights"])
def test_lengths(dev, dtype, R, weighted):
    q, kp, vp, table, n, g = _case(dev, R, EDGES, H=2, R=R, dtype=dtype, sharp=2.0)
    w = torch.rand(len(EDGES), table.shape[1] * R, generator=g, device=dev) if weighted else None
    out = _attend(q, kp, vp, table, n, w, what="lengths")
    assert (out[0] == 0).all()  # no cached row


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("T,G", [(1, 1), (1, 4), (3, 1), (5, 3), (16, 1), (17, 1), (33, 2), (64, 1), (65, 1), (130, 1)])
def test_query_rows_and_head_dims(dev, dtype, D, T, G):
    q, kp, vp, table, n, g = _case(dev, 7 * D + T, [300, 77, 1], H=3, G=G, D=D, R=32, T=T, dtype=dtype, sharp=1.5)
    w = torch.rand(3, table.shape[1] * 32, generator=g, device=dev)
    _attend(q, kp, vp, table, n, None, what="plain")
    _attend(q, kp, vp, table, n, w, what="weights")


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("lengths,T", [([45001], 1), ([20011, 3, 9999, 0, 12345], 2), ([6007] * 3, 40)])
def test_long_and_ragged(dev, dtype, lengths, T):
    q, kp, vp, table, n, g = _case(dev, T, lengths, R=64, T=T, dtype=dtype, slack=3, sharp=2.5)
    w = torch.zeros(len(lengths), table.shape[1] * 64, device=dev)
    _attend(q, kp, vp, table, n, None, what="long")
    _attend(q, kp, vp, table, n, w, what="long weights")
    # probabilities of every row sum to one
    total = w.double().sum(1)
    for i, length in enumerate(lengths):
        assert abs(float(total[i]) - (8 * T if length else 0)) < 1e-3 * 8 * T


@pytest.mark.parametrize("D,T,G,R", [(32, 7, 1, 64), (64, 13, 1, 16), (64, 20, 2, 256), (128, 25, 1, 32), (64, 70, 1, 64)])
def test_weights_of_many_query_rows(dev, D, T, G, R):
    # long caches and many query rows a head: the weights come from the keys once more; a page without rows, an infinite
    # key (which the padding of the query rows meets too), a NaN one, an empty sequence
    q, kp, vp, table, n, g = _case(dev, T, [33000, 1, 0, 20001], H=3, G=G, D=D, R=R, T=T, sharp=1.5)
    q = q.abs() + 0.1
    table[0, 5] = -1
    at = lambda s, r: (table[s, r // R].long(), slice(None), r % R)  # noqa: E731
    kp[at(0, 32000)] = float("-inf")
    w = torch.rand(4, table.shape[1] * R, generator=g, device=dev) * 0.01
    _attend(q, kp, vp, table, n, w, what="from the keys")
    assert torch.isfinite(w).all()
    kp[at(3, 7)] = float("nan")
    before = w.clone()
    import tabicl_mi355_paged as paged
    paged.paged_attention(q, kp, vp, table, n, w)
    assert torch.isnan(w[3, :20001]).all() and torch.equal(w[3, 20001:], before[3, 20001:])
    assert torch.isfinite(w[:3]).all()


def test_one_sequence_per_many(dev):
    # 300 sequences of a few rows
    q, kp, vp, table, n, g = _case(dev, 5, [(i * 7) % 40 for i in range(300)], H=1, R=16, T=2)
    _attend(q, kp, vp, table, n, torch.zeros(300, table.shape[1] * 16, device=dev), what="many")


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_pages_without_rows(dev, dtype):
    # page ids outside the pool inside and past the length, lengths below 0 and past the table
    q, kp, vp, table, n, g = _case(dev, 11, [200, 150, 90, 64], H=2, R=16, dtype=dtype, T=2)
    table[0, 3], table[0, 7], table[1, :] = -1, kp.shape[0], -5
    table[2, 0], table[2, 6:] = 2 ** 31 - 1, -1
    n[3] = -7
    w = torch.rand(4, table.shape[1] * 16, generator=g, device=dev)
    out = _attend(q, kp, vp, table, n, w, what="holes")
    assert (out[1] == 0).all() and (out[3] == 0).all()
    q, kp, vp, table, n, g = _case(dev, 12, [48, 48], H=2, R=16, dtype=dtype)
    want = _attend(q, kp, vp, table, n, what="full")
    n[:] = torch.tensor([2 ** 31 - 1, 49], dtype=torch.int32)  # clamped to the table
    assert torch.equal(_attend(q, kp, vp, table, n, what="past the table"), want)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_strided_views(dev, dtype):
    import tabicl_mi355_paged as paged
    N, H, T, D, R = 3, 4, 5, 64, 32
    q, kp, vp, table, n, g = _case(dev, 21, [100, 65, 33], H=H, T=T, R=R, dtype=dtype)
    want = _attend(q, kp, vp, table, n, what="contiguous")
    # heads of a projection, an unaligned view, a strided last dim, a broadcast query
    proj = torch.zeros(N, T, 3 * H * D, dtype=dtype, device=dev)
    proj.view(N, T, 3, H, D)[:, :, 1] = q.transpose(1, 2)
    odd = torch.zeros(q.numel() + 3, dtype=dtype, device=dev)[3:].view(q.shape).copy_(q)
    wide = torch.zeros(N, H, T, 2 * D, dtype=dtype, device=dev)[..., ::2].copy_(q)
    for view in (proj.view(N, T, 3, H, D)[:, :, 1].transpose(1, 2), odd, wide):
        assert torch.equal(paged.paged_attention(view, kp, vp, table, n), want)
    one = q[:1].expand(N, H, T, D)
    assert torch.equal(paged.paged_attention(one, kp, vp, table, n),
                       paged.paged_attention(one.contiguous(), kp, vp, table, n))
    # output in merged-head order, beside values that stay
    out = torch.full((N, T, H, 2 * D), 7.0, dtype=dtype, device=dev)
    o = paged.paged_attention(q, kp, vp, table, n, None, None, out[..., :D].transpose(1, 2))
    assert o.data_ptr() == out.data_ptr()
    assert torch.equal(out[..., :D].transpose(1, 2), want) and (out[..., D:] == 7).all()
    # a slice of a wider table, pages of a larger pool, weights with a row stride
    wide_t = torch.full((N, table.shape[1] + 4), -1, dtype=torch.int32, device=dev)
    wide_t[:, :table.shape[1]] = table
    big = torch.full((2, kp.shape[0], 3, *kp.shape[1:]), float("nan"), dtype=dtype, device=dev)
    big[0, :, 1], big[1, :, 2] = kp, vp
    w = torch.zeros(N, table.shape[1] * R + 9, device=dev)
    got = paged.paged_attention(q, big[0, :, 1], big[1, :, 2], wide_t[:, :table.shape[1]], n, w)
    assert torch.equal(got, want) and (w[:, table.shape[1] * R:] == 0).all()
    assert abs(float(w.sum()) - N * H * T) < 1e-2
    for bad in (torch.zeros(N, H, T, 2 * D, dtype=dtype, device=dev)[..., ::2],
                torch.zeros(N, 1, T, D, dtype=dtype, device=dev).expand(N, H, T, D)):
        with pytest.raises(ValueError, match="out needs"):
            paged.paged_attention(q, kp, vp, table, n, None, None, bad)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_non_finite_values(dev, dtype):
    # infinities and NaN in live rows reach what they should and nothing else
    lengths = [70, 70, 70, 70, 70, 700]
    q, kp, vp, table, n, g = _case(dev, 31, lengths, H=2, R=16, T=3, dtype=dtype)
    q = q.abs() + 0.1
    at = lambda s, r: (table[s, r // 16].long(), slice(None), r % 16)  # noqa: E731
    kp[at(0, 5)] = float("-inf")    # a key of score -inf: weight 0
    kp[at(1, 40)] = float("inf")    # a score of +inf: inf - inf
    kp[at(2, 69)] = float("nan")
    vp[at(3, 3)] = float("inf")
    vp[at(4, 64)] = float("nan")
    for r in range(600):            # whole tiles of -inf before the first finite score
        kp[at(5, r)] = float("-inf")
    w = torch.zeros(6, table.shape[1] * 16, device=dev)
    import tabicl_mi355_paged as paged
    out = paged.paged_attention(q, kp, vp, table, n, w)
    want, ww, tol, wtol = ref.attention(q, kp, vp, table, n, 0.125, torch.zeros_like(w))
    inf = torch.isinf(want)
    assert inf[3].all() and torch.equal(out.double()[inf], want[inf])
    ref.near(torch.where(inf, 0, out.double()), torch.where(inf, 0, want), torch.where(inf, 1, tol), "non-finite out")
    ref.near(w, ww, wtol, "non-finite weights")
    # every key at -inf: no weight anywhere, 0
    kp[table[0, :5].long()] = float("-inf")
    assert (paged.paged_attention(q, kp, vp, table, n)[0] == 0).all()


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("scale", [0.125, 4.0, -2.0, 0.0])
def test_sharp_scores(dev, dtype, scale):
    # scores that rise along the cache (every tile moves the running maximum) and fall along it, large scales
    q, kp, vp, table, n, g = _case(dev, 41, [3000, 3000], H=2, R=64, T=2, dtype=dtype)
    for s, sign in ((0, 1.0), (1, -1.0)):
        _, page, row = ref.rows_of(table[s], 3000, 64, kp.shape[0])
        kp[page, :, row] = (kp[page, :, row].float() + sign * torch.linspace(-4, 4, 3000, device=dev).view(-1, 1, 1)
                            ).to(dtype)
    q = (q.float().abs() * 0.5).to(dtype)
    _attend(q, kp, vp, table, n, torch.zeros(2, table.shape[1] * 64, device=dev), scale, "sharp")


def test_values_near_the_largest(dev):
    # fp32 values near the largest float survive the weighting; far negative scores with no others stay a softmax
    q, kp, vp, table, n, g = _case(dev, 43, [900, 40], H=1, R=16, T=1, dtype=F32)
    import tabicl_mi355_paged as paged
    vp[:] = torch.where(torch.isnan(vp), vp, torch.full_like(vp, 3e38))
    out = paged.paged_attention(q, kp, vp, table, n)
    assert torch.isfinite(out).all() and float((out / 3e38 - 1).abs().max()) < 1e-5
    _, page, row = ref.rows_of(table[1], 40, 16, kp.shape[0])
    kp[page, :, row] = -1e33
    q[1] = 1e3
    vp[page, :, row] = torch.arange(40.0, device=dev).view(40, 1, 1)
    assert torch.allclose(paged.paged_attention(q, kp, vp, table, n)[1], torch.tensor(19.5, device=dev))


def test_repeatable_and_concurrent(dev):
    # the same bits every time, on two streams at once and beside a default stream at work
    import tabicl_mi355_paged as paged
    q, kp, vp, table, n, g = _case(dev, 51, [9000, 4001, 200], T=4)
    w0 = torch.rand(3, table.shape[1] * 64, generator=g, device=dev)

    def once():
        w = w0.clone()
        return paged.paged_attention(q, kp, vp, table, n, w), w

    want = once()
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(once())
        got.append(once())
    torch.cuda.synchronize()
    for o, w in got:
        assert torch.equal(o, want[0]) and torch.equal(w, want[1])


def test_large_offsets(dev):
    # pages more than 2^32 elements apart in one pool
    import tabicl_mi355_paged as paged
    P, H, R, D = 2200, 8, 4096, 64  # 2200 x 2 Mi elements
    kp, vp = (torch.empty(P, H, R, D, dtype=BF, device=dev) for _ in range(2))
    ids = torch.tensor([[2199, 0], [2100, 2198]], dtype=torch.int32, device=dev)
    g = torch.Generator(device=dev).manual_seed(1)
    k, v = (torch.randn(2, H, 5000, D, generator=g, device=dev).to(BF) for _ in range(2))
    zero, n = (torch.tensor(x, dtype=torch.int32, device=dev) for x in ([0, 0], [5000, 5000]))
    paged.paged_append(kp, vp, ids, zero, k, v)
    for s in range(2):
        for t, want in ((kp, k), (vp, v)):
            got = torch.cat([t[ids[s, 0].long()], t[ids[s, 1].long(), :, :904]], 1)
            assert torch.equal(got, want[s])
    q = torch.randn(2, H, 2, D, generator=g, device=dev).to(BF)
    w = torch.zeros(2, 2 * R, device=dev)
    out = paged.paged_attention(q, kp, vp, ids, n, w)
    want, ww, tol, wtol = ref.attention(q, kp, vp, ids, n, D ** -0.5, torch.zeros_like(w))
    ref.near(out, want, tol, "far pages")
    ref.near(w, ww, wtol, "far pages weights")
    index, kw, kept = paged.paged_evict(kp, vp, ids, n, w, 4500, 16)
    assert kept.tolist() == [4500, 4500]
    for s in range(2):
        got = torch.cat([kp[ids[s, 0].long()], kp[ids[s, 1].long(), :, :404]], 1)
        assert torch.equal(got, k[s][:, index[s].long()])
    del kp, vp


# ---------------------------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("start,T", [([0, 0, 0], 1), ([5, 16, 31], 1), ([0, 7, 100], 77), ([90, 112, 200], 30), ([-3, 0, 1], 0)])
@pytest.mark.parametrize("counted", [False, True], ids=["", "count"])
def test_append(dev, dtype, D, start, T, counted):
    # starts inside a page, rows past the table dropped, pages the pool does not have dropped
    import tabicl_mi355_paged as paged
    H, R = 3, 16
    g = torch.Generator(device=dev).manual_seed(T + D)
    kp, vp = (torch.randn(30, H, R, D, generator=g, device=dev).to(dtype) for _ in range(2))
    table = torch.randperm(30, generator=g, device=dev)[:24].to(torch.int32).view(3, 8).contiguous()
    table[1, 2], table[2, 7] = -1, 30
    n = torch.tensor(start, dtype=torch.int32, device=dev)
    kv = torch.randn(3, T, 2, H, D, generator=g, device=dev).to(dtype)  # heads of a K|V projection
    k, v = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
    count = torch.tensor([T, T // 2, -1], dtype=torch.int32, device=dev) if counted else None
    want = ref.append(kp.cpu(), vp.cpu(), table.cpu(), n.cpu(), k.cpu(), v.cpu(), count)
    print(f"[paged] append {dtype} D={D} start={start} T={T} counted={counted}", flush=True)
    paged.paged_append(kp, vp, table, n, k, v, count)
    torch.cuda.synchronize()
    assert torch.equal(kp.cpu(), want[0]) and torch.equal(vp.cpu(), want[1]) and n.tolist() == start


def test_append_layouts(dev):
    # contiguous, unaligned and strided sources, a pool with gaps between its pages, a count past T
    import tabicl_mi355_paged as paged
    g = torch.Generator(device=dev).manual_seed(3)
    H, R, D, T = 2, 32, 64, 50
    k, v = (torch.randn(2, H, T, D, generator=g, device=dev).to(BF) for _ in range(2))
    table = torch.tensor([[4, 1], [0, 3]], dtype=torch.int32, device=dev)
    n = torch.tensor([3, 14], dtype=torch.int32, device=dev)
    odd = torch.zeros(k.numel() + 1, dtype=BF, device=dev)[1:].view(k.shape).copy_(k)
    wide = torch.zeros(2, H, T, 2 * D, dtype=BF, device=dev)[..., ::2].copy_(v)
    count = torch.tensor([1000, 50], dtype=torch.int32, device=dev)
    for a, b, c in ((k, v, None), (odd, wide, None), (k, wide, count)):
        pool = torch.full((5, 3, H, R, D), 9.0, dtype=BF, device=dev)
        kp, vp = pool[:, 0], pool[:, 2]
        want = ref.append(kp.cpu(), vp.cpu(), table.cpu(), n.cpu(), k.cpu(), v.cpu(), c)
        paged.paged_append(kp, vp, table, n, a, b, c)
        torch.cuda.synchronize()
        assert torch.equal(kp.cpu(), want[0]) and torch.equal(vp.cpu(), want[1]) and (pool[:, 1] == 9).all()


@pytest.mark.parametrize("dtype,D,R", [(BF, 64, 64), (F32, 32, 16), (BF, 128, 256), (F32, 128, 32)])
def test_gather(dev, dtype, D, R):
    # rows side by side; past the length (and past `rows`) nothing is written, a row without a page is 0
    import tabicl_mi355_paged as paged
    lengths = [0, 1, 100, 513, 300]
    q, kp, vp, table, n, g = _case(dev, D, lengths, H=3, R=R, D=D, dtype=dtype)
    table[3, 1] = -1
    for rows in (513, 200, 700, 0):
        k, v = paged.paged_gather(kp, vp, table, n, rows)
        marked = torch.full_like(k, 7.0), torch.full_like(v, 7.0)
        paged._gather_launch(kp, vp, table, n, *marked)
        torch.cuda.synchronize()
        assert k.shape == v.shape == (5, 3, rows, D)
        for s, length in enumerate(lengths):
            have = min(length, rows)
            at, page, row = ref.rows_of(table[s], have, R, kp.shape[0])
            for t, m, pages in ((k, marked[0], kp), (v, marked[1], vp)):
                want = torch.zeros(have, 3, D, dtype=dtype, device=dev)
                want[at] = pages[page, :, row]
                assert torch.equal(t[s, :, :have], want.transpose(0, 1)) and torch.equal(m[s, :, :have], want.transpose(0, 1))
                assert (m[s, :, have:] == 7).all()


# ---------------------------------------------------------------------------------------------
# eviction
# ---------------------------------------------------------------------------------------------
def _evict(kp, vp, table, n, w, keep, recent, what):
    import tabicl_mi355_paged as paged
    cpu = [t.cpu() for t in (kp, vp, table, n, w)]
    want = ref.evict(*cpu, keep.cpu() if torch.is_tensor(keep) else keep, recent)
    print(f"[paged] evict {what} pool {tuple(kp.shape)} keep {keep if not torch.is_tensor(keep) else keep.tolist()[:8]} "
          f"recent {recent}", flush=True)
    index, kw, kept = paged.paged_evict(kp, vp, table, n, w, keep, recent)
    torch.cuda.synchronize()
    assert torch.equal(kept.cpu(), want[4]), what
    assert torch.equal(index.cpu(), want[2]), what
    assert torch.equal(kw.cpu().view(torch.int32), want[3].view(torch.int32)), what
    for got, ref_pool in ((kp, want[0]), (vp, want[1])):
        assert torch.equal(got.cpu().view(torch.uint8), ref_pool.view(torch.uint8)), what
    for t, c in zip((table, n, w), cpu[2:]):  # read, not changed
        assert torch.equal(t.cpu().view(torch.int32), c.view(torch.int32))


LENGTHS = [0, 1, 2, 40, 63, 64, 65, 300, 1000, 1023, 1024, 1025, 2500]


@pytest.mark.parametrize("keep,recent", [(0, 0), (1, 0), (1, 5), (40, 0), (40, 7), (512, 32), (900, 900), (2499, 1), (2500, 0),
                                         (10000, 3)])
def test_evict(dev, keep, recent):
    q, kp, vp, table, n, g = _case(dev, keep + recent, LENGTHS, H=2, R=16, D=32, blocks=2)
    _evict(kp, vp, table, n, torch.exp(torch.randn(len(LENGTHS), table.shape[1] * 16, generator=g, device=dev) * 2), keep,
           recent, "log-normal")


@pytest.mark.parametrize("dtype,D,blocks", [(F32, 64, 1), (BF, 64, 3), (BF, 128, 1), (F32, 128, 2)])
def test_evict_types(dev, dtype, D, blocks):
    q, kp, vp, table, n, g = _case(dev, D, [700, 123, 64], H=3, R=64, D=D, dtype=dtype, blocks=blocks, slack=1)
    _evict(kp, vp, table, n, torch.rand(3, table.shape[1] * 64, generator=g, device=dev), 100, 10, "types")


def test_evict_ties_and_special_weights(dev):
    # equal weights, a few distinct ones, zeros of both signs, infinities, NaN, negative weights
    L = [1500] * 8
    q, kp, vp, table, n, g = _case(dev, 9, L, H=1, R=16, D=32, blocks=1)
    C = table.shape[1] * 16
    w = torch.zeros(8, C, device=dev)
    w[1] = 0.25
    w[2] = torch.randint(0, 3, (C,), generator=g, device=dev).float()
    w[3] = torch.where(torch.rand(C, generator=g, device=dev) < 0.5, -0.0, 0.0)
    w[4] = torch.randn(C, generator=g, device=dev)
    w[4, ::3], w[4, 1::7], w[4, 5::11] = float("nan"), float("inf"), float("-inf")
    w[5] = float("nan")
    w[6] = 1.0 + torch.arange(C, device=dev) * 2.0 ** -23  # neighbours in fp32, rising
    w[7] = torch.finfo(F32).tiny * 2.0 ** -10 * torch.randint(0, 2000, (C,), generator=g, device=dev)  # subnormal
    for keep, recent in ((1, 0), (700, 0), (700, 50), (1499, 0)):
        q, kp, vp, table, n, _ = _case(dev, 9, L, H=1, R=16, D=32, blocks=1)
        _evict(kp, vp, table, n, w, keep, recent, "ties")


def test_evict_budgets_and_layouts(dev):
    # a budget per sequence (negative and past the length too), weights with a row stride, one block without its dim,
    # pages the pool does not have, a pool whose blocks lie apart
    q, kp, vp, table, n, g = _case(dev, 13, [400, 400, 400, 50, 0], H=2, R=32, D=64)
    C = table.shape[1] * 32
    w = torch.rand(5, C + 5, generator=g, device=dev)[:, :C + 1]
    table[1, 2], table[2, 12] = -1, kp.shape[0]
    keep = torch.tensor([100, 399, 256, -4, 7], dtype=torch.int32, device=dev)
    import tabicl_mi355_paged as paged
    want = ref.evict(kp[None].cpu(), vp[None].cpu(), table.cpu(), n.cpu(), w.cpu(), keep.cpu(), 20)
    index, kw, kept = paged.paged_evict(kp, vp, table, n, w, keep, 20)
    torch.cuda.synchronize()
    assert index.shape == (5, C) and torch.equal(index.cpu(), want[2]) and torch.equal(kept.cpu(), want[4])
    assert torch.equal(kw.cpu(), want[3])
    for got, r in ((kp, want[0][0]), (vp, want[1][0])):
        assert torch.equal(got.cpu().view(torch.uint8), r.view(torch.uint8))
    pool = torch.randn(kp.shape[0], 3, 2, *kp.shape[1:], generator=g, device=dev).to(BF)
    _evict(pool[:, :, 0].transpose(0, 1), pool[:, :, 1].transpose(0, 1), table, n, w, 111, 0, "pages of all blocks")


@pytest.mark.parametrize("length,keep", [(70001, 30000), (45000, 44000)])
def test_evict_long(dev, length, keep):
    q, kp, vp, table, n, g = _case(dev, 17, [length, length // 3], H=1, R=256, D=32, blocks=1)
    w = torch.exp(torch.randn(2, table.shape[1] * 256, generator=g, device=dev))
    w = torch.where(torch.rand(w.shape, generator=g, device=dev) < 0.3, torch.zeros_like(w), w)
    _evict(kp, vp, table, n, w, keep, 100, "long")


# ---------------------------------------------------------------------------------------------
# graphs, ops, and the operators together
# ---------------------------------------------------------------------------------------------
def test_graph(dev):
    # one graph of append, attention with weights and eviction: replayed with other inputs, lengths and pages
    import tabicl_mi355_paged as paged
    q, kp, vp, table, n, g = _case(dev, 61, [3000, 900, 20], T=2, blocks=2, slack=2, spare=0)
    k, v = (torch.randn(3, 8, 10, 64, generator=g, device=dev).to(BF) for _ in range(2))
    w = torch.zeros(3, table.shape[1] * 64, device=dev)
    grown = n + 10

    def step():
        for b in range(2):
            paged.paged_append(kp[b], vp[b], table, n, k, v)
        out = paged.paged_attention(q, kp[0], vp[0], table, grown, w)
        return (out, *paged.paged_evict(kp, vp, table, grown, w, 800, 16))

    start = [t.clone() for t in (kp, vp, w)]

    def reset():
        for t, s in zip((kp, vp, w), start):
            t.copy_(s)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    with torch.cuda.graph(other):  # a second graph of the same calls, replayed between the first one's replays
        got2 = step()
    for i in range(3):
        q.copy_(torch.randn(q.shape, generator=g, device=dev).to(BF))
        k.copy_(torch.randn(k.shape, generator=g, device=dev).to(BF))
        n.copy_(torch.tensor([3000 - 700 * i, 900 + i, 20 * i], dtype=torch.int32))
        grown.copy_(n + 10)
        table.copy_(table.flip(0) if i == 1 else table)
        for t in start[:2]:
            t.copy_(torch.randn(t.shape, generator=g, device=dev).to(BF))
        results = []
        for run in (lambda: (graph.replay(), got)[1], lambda: (other.replay(), got2)[1], step):
            reset()
            torch.cuda.synchronize()
            r = run()
            torch.cuda.synchronize()
            results.append([t.clone() for t in (*r, kp, vp, w)])
        for a in results[:2]:
            for x, y in zip(a, results[2]):
                assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)), f"replay {i}"


def test_ops_equal_direct_calls(dev):
    import tabicl_mi355_paged as paged
    from torch.utils._python_dispatch import TorchDispatchMode

    class Seen(TorchDispatchMode):
        names: list = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.names.append(str(func))
            return func(*args, **(kwargs or {}))

    results = []
    for mode in (None, Seen()):
        q, kp, vp, table, n, g = _case(dev, 71, [500, 77], blocks=2)
        w = torch.zeros(2, table.shape[1] * 64, device=dev)
        out2 = torch.empty_like(q)

        def step():
            paged.paged_append(kp[1], vp[1], table, n - 3, q, q)
            out = paged.paged_attention(q, kp[1], vp[1], table, n, w)
            out1 = paged.paged_attention(q, kp[1], vp[1], table, n)
            paged.paged_attention(q, kp[0], vp[0], table, n, None, None, out2)
            return (out, out1, out2, w, *paged.paged_evict(kp, vp, table, n, w, 60, 3), kp, vp)

        if mode is None:
            results.append(step())
        else:
            with mode:
                results.append(step())
    for name in ("paged_append", "paged_attn.", "paged_attn_out", "paged_attn_weights_out", "paged_evict_out"):
        assert any(name in s for s in Seen.names), (name, Seen.names)
    for a, b in zip(*results):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_compile(dev):
    # torch.compile takes the wrappers as ops, whole graph, with their in-place results
    import tabicl_mi355_paged as paged
    q, kp, vp, table, n, g = _case(dev, 77, [300, 20], blocks=2)
    w = torch.rand(2, table.shape[1] * 64, generator=g, device=dev)
    start = [t.clone() for t in (kp, vp, w)]

    def step(q, kp, vp, table, n, w):
        paged.paged_append(kp[0], vp[0], table, n - 2, q, q)
        out = torch.zeros_like(q)
        paged.paged_attention(q * 2, kp[0], vp[0], table, n, w, None, out)
        index, kw, kept = paged.paged_evict(kp, vp, table, n, w, 50, 4)
        return out + 1, paged.paged_attention(q, kp[1], vp[1], table, kept), index, kw, kept

    want = [t.clone() for t in (*step(q, kp, vp, table, n, w), kp, vp, w)]
    for t, s in zip((kp, vp, w), start):
        t.copy_(s)
    got = (*torch.compile(step, fullgraph=True)(q, kp, vp, table, n, w), kp, vp, w)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_nothing_to_do(dev):
    # no sequences, no query rows, no pages in the table, an empty pool, nothing to keep
    import tabicl_mi355_paged as paged
    q, kp, vp, table, n, g = _case(dev, 79, [40, 5], H=2, R=16, T=2)
    assert paged.paged_attention(q[:0], kp, vp, table[:0], n[:0]).shape == (0, 2, 2, 64)
    assert paged.paged_attention(q[:, :, :0], kp, vp, table, n).shape == (2, 2, 0, 64)
    w = torch.rand(2, 48, generator=g, device=dev)
    before = w.clone()
    for pool, t in (((kp, vp), table[:, :0]), ((kp[:0], vp[:0]), table)):
        assert (paged.paged_attention(q, *pool, t, n, w) == 0).all()
        paged.paged_append(*pool, t, n, q, q)
    assert torch.equal(w, before)
    assert paged.paged_attention(q, kp, vp, table, n, w[:, :48], 0.1).shape == q.shape
    index, kw, kept = paged.paged_evict(kp, vp, table, n, w, 0)
    assert index.shape == (2, 0) and (kw == 0).all() and (kept == 0).all()
    index, kw, kept = paged.paged_evict(kp[None, :0].expand(3, -1, -1, -1, -1).contiguous(), vp[None, :0].expand(3, -1, -1, -1, -1).contiguous(),
                                        table, n, w, 7)
    assert kept.tolist() == [7, 5]
    index, kw, kept = paged.paged_evict(kp[None][:0], vp[None][:0], table, n, w, 7)
    assert kept.tolist() == [7, 5] and set(index[0].tolist()) == set(w[0, :40].topk(7).indices.tolist())
    torch.cuda.synchronize()


def test_gradient_refused(dev):
    import tabicl_mi355_paged as paged
    q, kp, vp, table, n, g = _case(dev, 73, [50])
    with pytest.raises(ValueError, match="no gradient"):
        paged.paged_attention(q.requires_grad_(), kp, vp, table, n)
    with torch.no_grad():
        paged.paged_attention(q, kp, vp, table, n)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_cache_together(dev, dtype):
    # tables of different sizes appended block by block, queried with the weights tracked, cut, grown and queried again:
    # what it answers is attention over the rows it says it holds
    import tabicl_mi355_paged as paged
    g = torch.Generator(device=dev).manual_seed(81)
    S, NB, H, D = 3, 2, 8, 64
    c = paged.PagedIclKVCache(S, NB, H, D, 1000, 40, 64, dtype, dev, track=True)
    c.keys.fill_(float("nan"))
    c.values.fill_(float("nan"))
    held = [[torch.zeros(0, H, D, dtype=dtype, device=dev)] * S for _ in range(2 * NB)]

    def grow(T, rows):
        for b in range(NB):
            k, v = (torch.randn(S, H, T, D, generator=g, device=dev).to(dtype) for _ in range(2))
            c.append(b, k, v, rows)
            for s in range(S):
                r = T if rows is None else rows[s]
                for i, x in ((2 * b, k), (2 * b + 1, v)):
                    held[i][s] = torch.cat([held[i][s], x[s, :, :r].transpose(0, 1)])

    def ask(T):
        before = c.weights.double().clone()
        total, tols = before.clone(), torch.zeros_like(before)
        for b in range(NB):
            q = (torch.randn(S, H, T, D, generator=g, device=dev) * 1.5).to(dtype)
            out = c.query(b, q)
            for s in range(S):
                k, v = held[2 * b][s], held[2 * b + 1][s]
                pool = [x.transpose(0, 1)[None].contiguous() for x in (k, v)]
                one = torch.zeros(1, 1, dtype=torch.int32, device=dev)
                n = torch.tensor([len(k)], dtype=torch.int32, device=dev)
                want, w, tol, wt = ref.attention(q[s:s + 1], *pool, one, n, D ** -0.5, torch.zeros(1, len(k), device=dev))
                ref.near(out[s:s + 1], want, tol, f"block {b} sequence {s}")
                total[s, :len(k)] += w[0]
                tols[s, :len(k)] += wt[0]
        ref.near(c.weights, total, tols + total.abs() * NB * 2.0 ** -23 + 2.0 ** -100, "tracked weights")

    grow(300, None)
    grow(400, [400, 100, 1])
    ask(1)
    ask(3)
    free = c.free_pages
    index = c.evict(256, recent=10)
    assert c.free_pages > free and [c.length(0, s) for s in range(S)] == [256, 256, 256]
    for i in range(2 * NB):
        held[i] = [held[i][s][index[s].long()] for s in range(S)]
    ask(2)
    grow(200, [200, 0, 100])
    ask(1)
    c.evict([300, 256, 1])
    c.release(1)
    assert [c.length(1, s) for s in range(S)] == [300, 0, 1]


@pytest.mark.parametrize("T", [2, 300])
def test_cache_query_in_a_graph(dev, T, monkeypatch):
    # a query captured once answers over the rows of the replay's time: more pages, fewer rows after an eviction
    import tabicl_mi355_paged as paged
    monkeypatch.setattr(paged, "_DENSE_SCORES", 1)
    g = torch.Generator(device=dev).manual_seed(85)
    c = paged.PagedIclKVCache(2, 1, 8, 64, 2000, 80, 64, BF, dev, track=T == 2)
    rows = lambda n: torch.randn(2, 8, n, 64, generator=g, device=dev).to(BF)  # noqa: E731
    c.append(0, rows(90), rows(90))
    q = rows(T)
    c.query(0, q)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = c.query(0, q)
    for step in range(3):
        if step < 2:
            c.append(0, rows(700), rows(700), [700, 300 * step])
        elif T == 2:
            c.evict(400)
        q.copy_(rows(T))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        k, v = paged.paged_gather(c.keys[0], c.values[0], c.table, c.lengths[0], c.capacity)
        for s in range(2):
            n = c.length(0, s)
            p = torch.softmax(q[s].double() @ k[s, :, :n].double().transpose(1, 2) / 8, -1)
            want = p @ v[s, :, :n].double()
            assert (out[s].double() - want).abs().max() <= 2.0 ** -8 * want.abs().max() + 1e-4, (step, s)


@pytest.mark.parametrize("valid", [None, 150])
def test_cache_many_query_rows(dev, valid, monkeypatch):
    # query rows by the hundred: gathered for the dense kernel, the same attention (to the bf16 bars: its probabilities are
    # bf16); an output view, an empty sequence, a valid length as a tensor; fewer rows and a tracked cache stay on the pages
    import tabicl_mi355_paged as paged
    from parity import check
    monkeypatch.setattr(paged, "_DENSE_SCORES", 1)
    gathers = []
    gather = paged.paged_gather
    monkeypatch.setattr(paged, "paged_gather", lambda *a: gathers.append(a[-1]) or gather(*a))
    g = torch.Generator(device=dev).manual_seed(83)
    for rows, track in (([700, 300, 65], False), ([700, 0, 65], False), ([700, 300, 65], True)):
        c = paged.PagedIclKVCache(3, 1, 8, 64, 800, 40, 64, BF, dev, track=track)
        k, v = (torch.randn(3, 8, 700, 64, generator=g, device=dev).to(BF) for _ in range(2))
        c.append(0, k, v, rows)
        q = torch.randn(3, 600, 8, 64, generator=g, device=dev).to(BF).transpose(1, 2)
        out = torch.zeros(3, 600, 8, 64, dtype=BF, device=dev)
        got = c.query(0, q, valid)
        c.query(0, q, valid, out.transpose(1, 2))
        torch.cuda.synchronize()
        assert torch.equal(out.transpose(1, 2), got)
        if valid is not None:
            assert torch.equal(c.query(0, q, torch.tensor([valid], device=dev)), got)
        for s, r in enumerate(rows):
            r = r if valid is None else min(r, valid)
            if r == 0:
                assert (got[s] == 0).all()
                continue
            p = torch.softmax(q[s].double() @ k[s, :, :r].double().transpose(1, 2) / 8, -1)
            check(got[s], p @ v[s, :, :r].double(), BF, f"sequence {s} of {rows}")
        c.query(0, q[:, :, :255], valid)
    assert gathers == ([700] * 4 if valid is None else [150, 150, 700] * 2)  # the untracked caches' calls


def test_cached_query_on_pages(dev):
    # the whole cached query of two tables on the paged cache against the dense one: the same rows, so logits as far
    # apart as two roundings of the bf16 attention output allow (parity.py's bf16 bars)
    import tabicl_mi355_icl as icl
    import tabicl_mi355_paged as paged
    import tabicl_mi355_query as Q
    from parity import check
    from query_ref import C, E, ICLH, NI, Rope, model, to_device
    w, g = model(F32)
    wd = to_device(w, dev)
    B, T, NF, train = 2, 3, 20, 600
    X = torch.randn(B, T, NF, generator=g).to(dev)
    col = Q.ColumnKVCache(3, B, NF + C, NI, E, F32, dev)
    for b in range(3):
        col.append_projected(b, torch.randn(B, NF + C, NI, E, generator=g).to(dev), wd.column.blocks[b])
    dense = icl.IclKVCache(B, 2, ICLH, train, 64, BF, dev)
    pages = paged.PagedIclKVCache(B, 2, ICLH, 64, 1024, 30, 64, BF, dev, track=True)
    for b in range(2):
        x = torch.randn(B, train, 512, generator=g).to(BF).to(dev)
        dense.append_projected(b, x, wd.icl_blocks[b].in_w, wd.icl_blocks[b].in_b)
        pages.append_projected(b, x[:, :400], wd.icl_blocks[b].in_w, wd.icl_blocks[b].in_b)
        pages.append_projected(b, x[:, 400:], wd.icl_blocks[b].in_w, wd.icl_blocks[b].in_b)
    for valid in (train, 250, torch.tensor([300], device=dev)):
        with torch.no_grad():
            want = Q.cached_query(X, None, col, dense, wd, valid, Rope())
            got = Q.cached_query(X, None, col, pages, wd, valid, Rope())
        torch.cuda.synchronize()
        check(got, want, BF, f"logits, valid {valid}", abs_tol=2e-2 * max(1.0, float(want.abs().max())))
    total = pages.weights.sum(1)
    assert torch.allclose(total, torch.full_like(total, 3 * 2 * ICLH * T), rtol=1e-4)
    with torch.no_grad():
        x = torch.randn(B, T, 512, generator=g).to(dev)
        a = pages.query_blocks(x, wd.icl_blocks)
        parts = pages.query_chunked(x, wd.icl_blocks, [(0, 1), (1, 2)])
    check(parts, a, BF, "chunked", abs_tol=2e-2 * max(1.0, float(a.abs().max())))


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("T,G", [(17, 1), (32, 1), (33, 1), (13, 5), (130, 1)])
def test_query_tiles_of_128_dims_on_long_caches(dev, dtype, T, G):
    # beyond 1,024 rows the query rows of a head go by 32 and 64 to a tile
    q, kp, vp, table, n, g = _case(dev, T, [1500, 0, 2777], H=2, G=G, D=128, R=64, T=T, dtype=dtype, slack=1, sharp=1.5)
    table[2, 3] = -1
    w = torch.rand(3, table.shape[1] * 64, generator=g, device=dev)
    _attend(q, kp, vp, table, n, None, what="tiles")
    _attend(q, kp, vp, table, n, w, what="tiles, weights")


@pytest.mark.parametrize("T,lengths", [(3, [300, 40]), (40, [9000, 17]), (70, [40000, 25001])])
def test_output_over_the_queries(dev, T, lengths):
    # in place, and shifted within one buffer; with the weights from the scores and from K again
    import tabicl_mi355_paged as paged
    q, kp, vp, table, n, g = _case(dev, T, lengths, H=4, T=T)
    w = [torch.zeros(2, table.shape[1] * 64, device=dev) for _ in range(3)]
    want = paged.paged_attention(q, kp, vp, table, n, w[0])
    for weights in (None, w[1]):
        buf = torch.zeros(2, 4, T + 1, 64, dtype=BF, device=dev)
        buf[:, :, 1:] = q
        for out in (buf[:, :, 1:], buf[:, :, :T]):
            buf[:, :, 1:] = q
            if weights is not None:
                weights.zero_()
            print(f"[paged] in place {T} {lengths} {weights is not None}", flush=True)
            assert paged.paged_attention(buf[:, :, 1:], kp, vp, table, n, weights, None, out) is out
            torch.cuda.synchronize()
            assert torch.equal(out, want)
            if weights is not None:
                assert torch.equal(weights, w[0])
    buf = q.clone()
    torch.ops.tabicl.paged_attn_weights_out(buf, kp, vp, table, n, 0.125, buf, w[2])
    torch.cuda.synchronize()
    assert torch.equal(buf, want) and torch.equal(w[2], w[0])


@pytest.mark.parametrize("dtype,D", [(BF, 64), (F32, 64), (BF, 128), (F32, 32)])
@pytest.mark.parametrize("H,G,T,lengths", [
    (8, 1, 1, [1999, 0, 5, 1030]), (1, 1, 32, [20000]), (1, 1, 33, [9000, 1]), (2, 8, 2, [1100, 4096]), (4, 1, 8, [128, 2048]),
    (1, 3, 1, [45000]), (2, 1, 1, [1500] * 70)])
def test_weights_of_few_rows(dev, dtype, D, H, G, T, lengths):
    # the references and sums joined where the weights are added up: items of one and of many parts, rows without a key,
    # up to 32 query rows a sequence and beyond
    q, kp, vp, table, n, g = _case(dev, T + H, lengths, H=H, G=G, D=D, T=T, dtype=dtype, sharp=2.0)
    w = torch.rand(len(lengths), table.shape[1] * 64 + 3, generator=g, device=dev)
    out = _attend(q, kp, vp, table, n, w, what="joined")
    again = torch.zeros_like(w), torch.zeros_like(w)
    import tabicl_mi355_paged as paged
    for x in again:
        assert torch.equal(paged.paged_attention(q, kp, vp, table, n, x), out)
    assert torch.equal(*again)


@pytest.mark.parametrize("seed,D,dtype,tracked", [(0, 64, BF, True), (1, 128, BF, True), (2, 32, F32, True), (3, 64, BF, False)])
def test_cache_through_random_calls(dev, seed, D, dtype, tracked):
    # appends, reservations, queries of many widths, evictions and releases in any order against lists of rows
    import random
    import tabicl_mi355_paged as paged
    S, B, H, R, cap = 4, 2, 2, 32, 2400
    rng, g = random.Random(seed), torch.Generator(device=dev).manual_seed(seed)
    c = paged.PagedIclKVCache(S, B, H, D, cap, 240, R, dtype, dev, track=tracked)
    for t in (c.keys, c.values):
        t.fill_(float("nan"))
    rows = [[(torch.empty(H, 0, D, dtype=dtype, device=dev),) * 2 for _ in range(S)] for _ in range(B)]
    for step in range(60):
        have = [rows[0][s][0].shape[1] for s in range(S)]
        what = rng.choice(["append", "append", "query", "query", "query", "evict", "release", "reserve", "captured"])
        print(f"[paged] step {step} {what} {have} free {c.free_pages}", flush=True)
        if what == "append":
            T = rng.choice([1, 7, 33, 400, 1500])
            new = [rng.choice([0, T, rng.randint(0, T)]) for _ in range(S)]
            new = [min(n, cap - h) for n, h in zip(new, have)]
            if sum(max(c._held[s], -(-(h + n) // R)) - c._held[s] for s, (h, n) in enumerate(zip(have, new))) > c.free_pages:
                with pytest.raises(ValueError, match="pages wanted"):
                    c.append(0, *(torch.zeros(S, H, T, D, dtype=dtype, device=dev),) * 2, new)
                continue
            for b in range(B):
                k, v = (torch.randn(S, T, H, D, generator=g, device=dev).to(dtype).transpose(1, 2) for _ in range(2))
                c.append(b, k, v, new)
                for s in range(S):
                    rows[b][s] = tuple(torch.cat([o, x[s, :, :new[s]]], 1) for o, x in zip(rows[b][s], (k, v)))
        elif what in ("query", "captured") and max(have):
            b, T = rng.randrange(B), rng.choice([1, 3, 20, 70])
            q = torch.randn(S, H, T, D, generator=g, device=dev).to(dtype)
            before = None if c.weights is None else c.weights.clone()
            want, w, tol, wtol = ref.attention(q, c.keys[b], c.values[b], c.table, c.lengths[b], D ** -0.5, before)
            if what == "query":
                out = c.query(b, q, None, rng.choice([None, torch.empty_like(q), q]))
            else:
                c.query(b, q)
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    out = c.query(b, q)
                for _ in range(2):
                    if before is not None:
                        c.weights.copy_(before)
                    graph.replay()
            torch.cuda.synchronize()
            ref.near(out, want, tol, "out")
            if before is not None:
                ref.near(c.weights, w, wtol, "weights")
        if what == "evict" and tracked:
            keep = rng.choice([rng.randint(0, 2000), [rng.randint(0, 2000) for _ in range(S)]])
            recent = rng.choice([0, 5, 3000])
            before = c.weights.clone()
            index = c.evict(keep, recent).long()
            for s in range(S):
                n = min(have[s], keep if isinstance(keep, int) else keep[s])
                idx, last = index[s, :n], min(recent, n)
                assert (index[s, n:] == -1).all() and len(set(idx.tolist())) == n
                assert set(range(have[s] - last, have[s])) <= set(idx.tolist())
                assert torch.equal(c.weights[s, :n], before[s, idx]) and (c.weights[s, n:] == 0).all()
                gone = torch.ones(have[s] - last, dtype=torch.bool, device=dev)  # of the rows that compete
                gone[idx[idx < have[s] - last]] = False
                older = before[s, :have[s] - last]
                assert not gone.any() or gone.all() or older[gone].max() <= older[~gone].min()
                for b in range(B):
                    rows[b][s] = tuple(x[:, idx] for x in rows[b][s])
        elif what == "release":
            s = rng.randrange(S)
            c.release(s)
            for b in range(B):
                rows[b][s] = tuple(x[:, :0] for x in rows[b][s])
        elif what == "reserve":
            want = [rng.randint(0, 600) for _ in range(S)]
            if sum(max(0, -(-n // R) - held) for n, held in zip(want, c._held)) <= c.free_pages:
                c.reserve(want)
        # the books, and what the pages hold
        assert c.free_pages + sum(c._held) == 240
        table = c.table.tolist()
        owned = [p for t in table for p in t if p >= 0]
        assert len(set(owned)) == len(owned) == sum(c._held)
        for b in range(B):
            assert c.lengths[b].tolist() == [rows[b][s][0].shape[1] for s in range(S)]
            for s in range(S):
                n = c.length(b, s)
                _, page, row = ref.rows_of(c.table[s], n, R, 240)
                for pool, want in zip((c.keys, c.values), rows[b][s]):
                    assert torch.equal(pool[b][page, :, row].transpose(0, 1), want)


@pytest.mark.parametrize("size", [1e6, 1e8, 1e10])
@pytest.mark.parametrize("T,lengths", [(13, [40000, 25600]), (70, [65000, 700])])
def test_weights_of_large_scores(dev, size, T, lengths):
    # weights from the keys once more, products q.K of `size`: every query row's probabilities sum to one, and they are
    # those of the same rows twelve at a time, which come from stored scores. Both take the same bf16 products; a
    # probability's rounding errors are the exponential's, the sums' over the keys (n / 32 + 128 steps) and the
    # normaliser's, the weights' those of one addition per query row.
    import tabicl_mi355_paged as paged
    q, kp, vp, table, n, g = _case(dev, T, lengths, H=2, T=T)
    q = (q.float() * size ** 0.5).to(BF)
    kp *= size ** 0.5
    w, few = torch.zeros(2, table.shape[1] * 64, device=dev), torch.zeros(2, table.shape[1] * 64, device=dev)
    assert w.numel() >= 65536
    print(f"[paged] large scores {size} {T} {lengths}", flush=True)
    out = paged.paged_attention(q, kp, vp, table, n, w)
    for t in range(0, T, 12):
        paged.paged_attention(q[:, :, t:t + 12], kp, vp, table, n, few)
    torch.cuda.synchronize()
    assert torch.isfinite(out).all() and torch.isfinite(w).all()
    for s, length in enumerate(lengths):
        e = (length / 32 + 128 + 2 * T + 16) * 2.0 ** -24
        assert abs(float(w[s].double().sum()) / (2 * T) - 1) <= e
        diff = (w[s].double() - few[s].double()).abs()
        assert bool((diff <= 2 * e * few[s].double() + 2.0 ** -100).all()), float((diff / few[s].clamp(min=1e-30)).max())


@pytest.mark.parametrize("H,G,D,T,lengths,dtype", [
    (8, 1, 64, 12001, [3000], BF), (8, 1, 64, 2500, [7000, 33], F32), (2, 3, 128, 5000, [1000, 0, 5000], F32),
    (1, 5, 32, 14000, [4000], F32)])
def test_weights_of_query_rows_in_slices(dev, H, G, D, T, lengths, dtype):
    # more scores than are kept at a time: slices of the query rows, the last one shorter; the rows of an output view
    import tabicl_mi355_native as nat
    import tabicl_mi355_paged as paged
    q, kp, vp, table, n, g = _case(dev, T, lengths, H=H, G=G, D=D, T=T, dtype=dtype)
    N, rows = len(lengths), table.shape[1] * 64
    assert N * H * G * T * rows * 4 > 1 << 30
    assert nat.load().tabicl_paged_attn_workspace_bytes(N, H * G, H, T, D, rows, 1, int(dtype is F32)) < 1152 << 20
    w = torch.rand(N, rows, generator=g, device=dev)
    w0, w1 = w.clone(), w.clone()
    want = _attend(q, kp, vp, table, n, w, what="slices")
    merged = torch.empty(N, T, H * G, D, dtype=dtype, device=dev)
    proj = torch.empty(N, T, H * G, D, dtype=dtype, device=dev).copy_(q.transpose(1, 2))
    paged.paged_attention(proj.transpose(1, 2), kp, vp, table, n, w0, None, merged.transpose(1, 2))
    torch.cuda.synchronize()
    assert torch.equal(merged.transpose(1, 2), want) and torch.equal(w0, w)
    paged.paged_attention(q, kp, vp, table, n, w1, None, q)  # over the queries
    torch.cuda.synchronize()
    assert torch.equal(q, want) and torch.equal(w1, w)


@pytest.mark.parametrize("lengths,weighted", [([200, 3, 0, 64, 17, 100, 1, 128], True), ([1100] + [5] * 7, False)])
def test_query_rows_beyond_one_launch(dev, lengths, weighted):
    # more than 2^22 query rows over all sequences and heads
    T = 66000
    q, kp, vp, table, n, g = _case(dev, 3, lengths, H=8, D=32, T=T)
    assert 8 * 8 * T > 1 << 22
    w = torch.zeros(8, table.shape[1] * 64, device=dev) if weighted else None
    _attend(q, kp, vp, table, n, w, what="many rows")


def test_cache_many_query_rows_of_ragged_tables(dev, monkeypatch):
    # the gathered rows in runs of sequences: the same attention as all at once, whichever sequences share a run
    import tabicl_mi355_paged as paged
    from parity import check
    monkeypatch.setattr(paged, "_DENSE_SCORES", 1)
    lengths = [40, 3000, 0, 700, 1, 5000, 64, 129]
    c = paged.PagedIclKVCache(8, 1, 8, 64, 5000, 150, 64, BF, dev)
    g = torch.Generator(device=dev).manual_seed(87)
    k, v = (torch.randn(8, 8, 5000, 64, generator=g, device=dev).to(BF) for _ in range(2))
    c.append(0, k, v, lengths)
    q = torch.randn(8, 300, 8, 64, generator=g, device=dev).to(BF).transpose(1, 2)
    for rows in (1, 1500, 8000):
        monkeypatch.setattr(paged, "_GATHER_BYTES", rows * 2 * 8 * 64 * 2)
        got, out = c.query(0, q), torch.zeros(8, 300, 8, 64, dtype=BF, device=dev)
        c.query(0, q, None, out.transpose(1, 2))
        over = q.clone()
        c.query(0, over, None, over)
        torch.cuda.synchronize()
        assert torch.equal(out.transpose(1, 2), got) and torch.equal(over, got)
        for s, n in enumerate(lengths):
            if n == 0:
                assert (got[s] == 0).all()
            else:
                p = torch.softmax(q[s].double() @ k[s, :, :n].double().transpose(1, 2) / 8, -1)
                check(got[s], p @ v[s, :, :n].double(), BF, f"sequence {s}, runs of {rows} rows")


def test_cache_many_query_rows_of_grouped_heads(dev, monkeypatch):
    # groups of query heads stay on the pages at any number of rows
    import tabicl_mi355_paged as paged
    monkeypatch.setattr(paged, "_DENSE_SCORES", 1)
    c = paged.PagedIclKVCache(2, 1, 2, 64, 2000, 40, 64, BF, dev)
    g = torch.Generator(device=dev).manual_seed(89)
    k, v = (torch.randn(2, 2, 1100, 64, generator=g, device=dev).to(BF) for _ in range(2))
    c.append(0, k, v, [1100, 90])
    q = torch.randn(2, 6, 600, 64, generator=g, device=dev).to(BF)
    want, _, tol, _ = ref.attention(q, c.keys[0], c.values[0], c.table, c.lengths[0], 0.125)
    ref.near(c.query(0, q), want, tol, "grouped heads")


@pytest.mark.parametrize("T", [3, 400])
def test_cache_chunks_of_empty_tables(dev, T, monkeypatch):
    # query_chunked over chunks with and without rows equals one query over all of them
    import tabicl_mi355_icl as icl
    import tabicl_mi355_paged as paged
    monkeypatch.setattr(paged, "_DENSE_SCORES", 1)
    g = torch.Generator(device=dev).manual_seed(91)
    r = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    blocks = [icl.IclBlockWeights(r(512), r(512), (r(1536, 512) / 22).to(BF), None, (r(512, 512) / 22).to(BF), None, r(512), r(512),
                                  (r(1024, 512) / 22).to(BF), None, (r(512, 1024) / 32).to(BF), None) for _ in range(2)]
    c = paged.PagedIclKVCache(4, 2, 8, 64, 300, 30, 64, BF, dev)
    for b in range(2):
        c.append(b, r(4, 8, 300, 64).to(BF), r(4, 8, 300, 64).to(BF), [300, 0, 50, 0])
    c.release(2)
    x = r(4, T, 512)
    with torch.no_grad():
        want = c.query_blocks(x, blocks)
        for chunks in ([(0, 1), (1, 2), (2, 4)], [(0, 2), (2, 3), (3, 4)]):
            got = c.query_chunked(x, blocks, chunks)
            torch.cuda.synchronize()
            assert torch.allclose(got, want, rtol=2.0 ** -6, atol=2.0 ** -6 * float(want.abs().max()))
            assert torch.isfinite(got).all()


@pytest.mark.parametrize("T", [2, 300])
def test_cache_query_with_a_limit_in_a_graph(dev, T, monkeypatch):
    # a number for valid_kv_len holds in every replay, also where the cache was shorter when the query was captured
    import tabicl_mi355_paged as paged
    monkeypatch.setattr(paged, "_DENSE_SCORES", 1)
    g = torch.Generator(device=dev).manual_seed(93)
    c = paged.PagedIclKVCache(2, 1, 8, 64, 1000, 40, 64, BF, dev, track=T == 2)
    rows = lambda n: torch.randn(2, 8, n, 64, generator=g, device=dev).to(BF)  # noqa: E731
    c.append(0, rows(90), rows(90), [90, 60])
    q = rows(T)
    for limit in (200, 250, 75, 10 ** 12, 0):
        c.query(0, q, limit)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = c.query(0, q, limit)
        c.append(0, rows(150), rows(150), [150, 20])
        for _ in range(2):
            q.copy_(rows(T))
            before = None if c.weights is None else c.weights.clone()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            n = c.lengths[0].clamp(max=min(limit, 1000))
            want, w, tol, wtol = ref.attention(q, c.keys[0], c.values[0], c.table, n, 0.125, before)
            ref.near(out, want, tol, f"limit {limit}")
            if before is not None:
                ref.near(c.weights, w, wtol, f"limit {limit}, weights")


def test_cache_books_refuse_capture(dev):
    # calls that keep books on the host are refused while a graph is captured, and change nothing
    import tabicl_mi355_paged as paged
    c = paged.PagedIclKVCache(2, 1, 8, 64, 500, 20, 64, BF, dev, track=True)
    z = torch.zeros(2, 8, 10, 64, dtype=BF, device=dev)
    c.append(0, z, z)
    c.reserve(500)  # an append needs no page: nothing else would stop it
    q = torch.ones(2, 8, 1, 64, dtype=BF, device=dev)
    c.query(0, q)
    before = [t.clone() for t in (c.table, c.lengths, c.weights)], c.free_pages
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = c.query(0, q)
        for call in (lambda: c.append(0, z, z), lambda: c.append(0, z, z, [1, 0]), lambda: c.evict(4), lambda: c.release(0),
                     lambda: c.reserve(20)):
            with pytest.raises(ValueError, match="captured"):
                call()
    assert c.length(0, 0) == c.length(0, 1) == 10 and c.free_pages == before[1]
    for t, b in zip((c.table, c.lengths, c.weights), before[0]):
        assert torch.equal(t, b)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, c.query(0, q))


def test_query_blocks_refuse_gradients(dev):
    # of the rows and of any weight, in both modes: the layers between the attentions would drop them without a word
    import torch.autograd.forward_ad as fw
    import dataclasses
    import tabicl_mi355_icl as icl
    import tabicl_mi355_paged as paged
    g = torch.Generator(device=dev).manual_seed(95)
    r = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    blocks = [icl.IclBlockWeights(r(512), r(512), (r(1536, 512) / 22).to(BF), None, (r(512, 512) / 22).to(BF), None, r(512), r(512),
                                  (r(1024, 512) / 22).to(BF), None, (r(512, 1024) / 32).to(BF), None) for _ in range(2)]
    c = paged.PagedIclKVCache(1, 2, 8, 64, 100, 4, 64, BF, dev)
    for b in range(2):
        c.append(b, r(1, 8, 100, 64).to(BF), r(1, 8, 100, 64).to(BF))
    x = r(1, 5, 512)
    want = c.query_blocks(x, blocks)
    for name in (None, "ln1_w", "in_w", "out_w", "ln2_b", "ff2_w"):
        other = blocks if name is None else [dataclasses.replace(blocks[0], **{name: getattr(blocks[0], name).clone().requires_grad_()}),
                                             blocks[1]]
        y = x.clone().requires_grad_() if name is None else x
        with pytest.raises(ValueError, match="no gradient"):
            c.query_blocks(y, other)
        with pytest.raises(ValueError, match="no gradient"):
            c.query_chunked(y, other, [(0, 1)])
        with torch.no_grad():
            assert torch.equal(c.query_blocks(y, other), want)
    with fw.dual_level(), pytest.raises(ValueError, match="no gradient"):
        c.query_blocks(fw.make_dual(x, torch.ones_like(x)), blocks)


@pytest.mark.parametrize("keep,recent", [(2 ** 64 + 5, 0), (10, 2 ** 64 + 1), (2 ** 63, 2 ** 63)])
def test_evict_with_numbers_beyond_64_bits(dev, keep, recent):
    # no limit, and all rows recent: not what is left of the number in 64 bits
    q, kp, vp, table, n, g = _case(dev, 19, [40, 0, 64], H=2, R=16, D=32, blocks=2)
    w = torch.rand(3, table.shape[1] * 16, generator=g, device=dev)
    _evict(kp, vp, table, n, w, keep, recent, "huge numbers")


@pytest.mark.parametrize("lengths,keep,recent", [([300001, 5], 292000, 40000), ([262145, 262144, 600000], 262100, 3),
                                                 ([530000], 520000, 0)])
def test_evict_of_very_long_sequences(dev, lengths, keep, recent):
    # beyond 262,144 rows a workgroup ranks several blocks of 1,024 rows: many ties at the threshold, recent rows from the
    # middle of a block on
    q, kp, vp, table, n, g = _case(dev, 23, lengths, H=1, R=256, D=32, blocks=1)
    w = torch.randint(0, 40, (len(lengths), table.shape[1] * 256), generator=g, device=dev).float()
    _evict(kp, vp, table, n, w, keep, recent, "very long")


def test_evict_time_grows_with_the_rows(dev):
    # four times the rows in about four times the time, not sixteen (twice the linear time is allowed)
    import tabicl_mi355_paged as paged

    def us(rows):
        pool = torch.zeros(1, 1, 1, 1024, 32, dtype=BF, device=dev)
        table = torch.full((1, rows // 1024), -1, dtype=torch.int32, device=dev)  # the ranks' time, without moves
        n = torch.tensor([rows], dtype=torch.int32, device=dev)
        w = torch.rand(1, rows, device=dev)
        best = float("inf")
        for _ in range(4):
            start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            start.record()
            paged.paged_evict(pool, pool.clone(), table, n, w, 16)
            end.record()
            torch.cuda.synchronize()
            best = min(best, start.elapsed_time(end) * 1e3)
        return best

    few, many = us(1 << 22), us(1 << 24)
    print(f"[paged] eviction of 2^22 rows {few:.0f} us, of 2^24 {many:.0f}", flush=True)
    assert many < 8 * few


@pytest.mark.parametrize("D,T,L", [(64, 4, 1381), (64, 24, 300), (128, 4, 1700), (128, 40, 2100), (32, 4, 40), (64, 2, 5)])
@pytest.mark.parametrize("sharp", [0.5, 3.0])
def test_fp32_accuracy(dev, D, T, L, sharp):
    # In the 2-norm as near to float64 as scores whose products are summed in fp32 in four chains, with everything after them
    # in float64: that is the rounding that cannot be avoided without more bits. A quarter on top for the chains' order, and
    # 2^-23 for the exponential (one unit), the sums over the keys and the output's own rounding.
    q, kp, vp, table, n, g = _case(dev, D + T, [L] * 4, D=D, T=T, dtype=F32, sharp=sharp)
    import tabicl_mi355_paged as paged
    w = torch.zeros(4, table.shape[1] * 64, device=dev)
    out = paged.paged_attention(q, kp, vp, table, n, w)
    want, ww, _, _ = ref.attention(q, kp, vp, table, n, D ** -0.5, torch.zeros_like(w))
    four, fw = torch.zeros_like(want), torch.zeros_like(ww)
    for s in range(4):
        at, page, row = ref.rows_of(table[s], L, 64, kp.shape[0])
        k, v = (t[page, :, row].transpose(0, 1).double() for t in (kp, vp))  # [H, L, D]
        parts = []
        for c in range(4):
            acc = torch.zeros(8, T, L, device=dev)
            for d in range(c, D, 4):
                acc = (acc.double() + q[s, :, :, d, None].double() * k[:, None, :, d]).float()
            parts.append(acc)
        x = ((parts[0] + parts[1]) + (parts[2] + parts[3])).double()
        p = torch.softmax(x * D ** -0.5, -1)
        four[s], fw[s, :L] = torch.matmul(p, v), p.sum((0, 1))
    for name, a, b, c in (("out", out, want, four), ("weights", w, ww, fw)):
        err, least = (float((t.double() - b).norm() / b.norm()) for t in (a, c))
        print(f"[paged] fp32 {name} D={D} T={T} L={L} sharp {sharp}: {err:.2e}, four chains {least:.2e}", flush=True)
        assert err <= 1.25 * least + 2.0 ** -23, name


@pytest.mark.parametrize("seed", range(24))
def test_random_cases(dev, seed):
    # types, head layouts, page sizes, lengths, missing pages, weights, appends and budgets at random
    import random
    import tabicl_mi355_paged as paged
    rng = random.Random(seed)
    dtype, D, R = rng.choice([BF, F32]), rng.choice([32, 64, 128]), 1 << rng.randint(4, 9)
    H, G, N = rng.choice([1, 2, 3, 8]), rng.choice([1, 1, 2, 5]), rng.choice([1, 2, 3, 7, 65, 130])
    top = rng.choice([40, 1024, 1500, 6000, 20000]) if N < 8 else rng.choice([40, 300, 1500])
    edges = [0, 1, 15, 16, 17, 127, 128, 129, 255, 256, 257, 1023, 1024, 1025, 2047, 2049]
    lengths = [min(top, rng.choice(edges) if rng.random() < 0.3 else rng.randint(0, top)) for _ in range(N)]
    T = rng.choice([1, 1, 2, 5, 17, 40, 70])
    if max(lengths) * N * H * G * T > 3e7:
        T = 1
    q, kp, vp, table, n, g = _case(dev, seed, lengths, H=H, G=G, D=D, R=R, T=T, dtype=dtype, slack=rng.choice([0, 0, 3]),
                                   sharp=rng.choice([0.3, 1.0, 4.0]))
    whole = table.clone()
    if rng.random() < 0.3:
        gone = torch.randint(0, table.numel(), (max(1, table.numel() // 6),), generator=g, device=dev)
        table.view(-1)[gone] = rng.choice([-1, kp.shape[0], 1 << 30])
    w = torch.rand(N, table.shape[1] * R, generator=g, device=dev) * 0.1 if rng.random() < 0.6 else None
    _attend(q, kp, vp, table, n, w, what=f"random {seed}")
    if kp.numel() > 3e7:
        return
    new = rng.randint(1, 60)
    k, v = (torch.randn(N, H, new, D, generator=g, device=dev).to(dtype) for _ in range(2))
    want = ref.append(kp.cpu(), vp.cpu(), whole.cpu(), n.cpu(), k.cpu(), v.cpu())
    paged.paged_append(kp, vp, whole, n, k, v)
    torch.cuda.synchronize()
    for got, x in zip((kp, vp), want):
        assert torch.equal(got.cpu().view(torch.uint8), x.view(torch.uint8))
    shape = (N, table.shape[1] * R)
    weights = rng.choice([lambda: torch.rand(shape, generator=g, device=dev),
                          lambda: torch.randint(0, 4, shape, generator=g, device=dev).float(),
                          lambda: torch.exp(torch.randn(shape, generator=g, device=dev) * 20)])()
    keep = rng.choice([rng.randint(0, top), torch.randint(-2, top + 5, (N,), generator=g, device=dev, dtype=torch.int32)])
    _evict(kp[None], vp[None], whole, n, weights, keep, rng.choice([0, 0, 3, top]), f"random {seed}")


def test_slices_in_a_graph(dev):
    # a call that goes in slices, captured: every replay adds its weights once
    import tabicl_mi355_paged as paged
    q, kp, vp, table, n, g = _case(dev, 97, [3000], H=8, T=12001)
    w = torch.zeros(1, table.shape[1] * 64, device=dev)
    paged.paged_attention(q, kp, vp, table, n, w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged.paged_attention(q, kp, vp, table, n, w)
    for step in range(3):
        q.copy_(torch.randn(q.shape, generator=g, device=dev).to(BF))
        n.fill_(3000 - 700 * step)
        w.zero_()
        want = paged.paged_attention(q, kp, vp, table, n, w)
        ww = w.clone()
        w.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(w, ww), step
