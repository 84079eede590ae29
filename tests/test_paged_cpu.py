"""CPU tests of the paged K/V cache: what the wrappers and the C ABI refuse, and PagedIclKVCache's books (pages, lengths,
weights) with the plain forms in the kernels' place."""
import pytest
import torch

import paged_ref as ref


def _pool(P=6, H=2, R=16, D=64, dtype=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed)
    return tuple(torch.randn(P, H, R, D, generator=g).to(dtype) for _ in range(2))


def _table(N=2, M=3):
    return torch.arange(N * M, dtype=torch.int32).view(N, M)


def test_no_cpu_path():
    import tabicl_mi355_native as nat
    import tabicl_mi355_paged as paged
    k, v = _pool()
    t, n, q = _table(), torch.tensor([5, 9], dtype=torch.int32), torch.randn(2, 2, 1, 64)
    with pytest.raises(nat.NativeLibraryError):
        paged.paged_attention(q, k, v, t, n)
    with pytest.raises(nat.NativeLibraryError):
        paged.paged_append(k, v, t, n, q, q)
    with pytest.raises(nat.NativeLibraryError):
        paged.paged_evict(k, v, t, n, torch.zeros(2, 48), 4)
    with pytest.raises(nat.NativeLibraryError):
        paged.paged_gather(k, v, t, n, 9)
    for bad in ((k[0], v[0], t, n, 9), (k, v, t, n, -1), (k, v[:2], t, n, 9), (k, v, t.long(), n, 9)):
        with pytest.raises(ValueError):
            paged.paged_gather(*bad)


@pytest.mark.parametrize("change,word", [
    (dict(q=torch.zeros(2, 3, 1, 64)), "multiple of 2 heads"),
    (dict(q=torch.zeros(3, 2, 1, 64)), "must be"),
    (dict(q=torch.zeros(2, 2, 1, 32)), "must be"),
    (dict(q=torch.zeros(2, 2, 64)), "must be"),
    (dict(q=torch.zeros(2, 2, 1, 64, dtype=torch.bfloat16)), "cast q"),
    (dict(table=torch.zeros(2, 3, dtype=torch.int64)), "int32"),
    (dict(table=torch.zeros(6, dtype=torch.int32)), "int32"),
    (dict(lengths=torch.zeros(2, dtype=torch.int64)), "lengths"),
    (dict(lengths=torch.zeros(3, dtype=torch.int32)), "lengths"),
    (dict(v=torch.zeros(6, 2, 16, 32)), "one layout"),
    (dict(k=torch.zeros(6, 16, 2, 64).transpose(1, 2), v=torch.zeros(6, 16, 2, 64).transpose(1, 2)), "contiguous"),
    (dict(weights=torch.zeros(2, 47)), "weights"),
    (dict(weights=torch.zeros(2, 48, dtype=torch.float64)), "weights"),
    (dict(weights=torch.zeros(48, 2).t()), "weights"),
    (dict(out=torch.zeros(2, 2, 2, 64)), "out"),
    (dict(q=torch.zeros(2, 2, 1, 64, requires_grad=True)), "no gradient"),
])
def test_attention_refuses(change, word):
    import tabicl_mi355_paged as paged
    k, v = _pool()
    a = dict(q=torch.zeros(2, 2, 1, 64), k=k, v=v, table=_table(), lengths=torch.tensor([5, 9], dtype=torch.int32),
             weights=None, out=None)
    a.update(change)
    with pytest.raises(ValueError, match=word):
        paged.paged_attention(a["q"], a["k"], a["v"], a["table"], a["lengths"], a["weights"], None, a["out"])


@pytest.mark.parametrize("change,word", [
    (dict(k=torch.zeros(2, 2, 4, 32), v=torch.zeros(2, 2, 4, 32)), "must be"),
    (dict(v=torch.zeros(2, 2, 3, 64)), "must be"),
    (dict(k=torch.zeros(2, 2, 4, 64, dtype=torch.bfloat16)), "cast"),
    (dict(count=torch.zeros(2, dtype=torch.int64)), "count"),
    (dict(count=torch.zeros(1, dtype=torch.int32)), "count"),
    (dict(k=torch.zeros(2, 2, 4, 64, requires_grad=True)), "no gradient"),
])
def test_append_refuses(change, word):
    import tabicl_mi355_paged as paged
    kp, vp = _pool()
    a = dict(k=torch.zeros(2, 2, 4, 64), v=torch.zeros(2, 2, 4, 64), count=None)
    a.update(change)
    with pytest.raises(ValueError, match=word):
        paged.paged_append(kp, vp, _table(), torch.zeros(2, dtype=torch.int32), a["k"], a["v"], a["count"])


@pytest.mark.parametrize("change,word", [
    (dict(keep=-1), "negative"),
    (dict(recent=-1), "negative"),
    (dict(keep=torch.zeros(3, dtype=torch.int32)), "keep"),
    (dict(keep=torch.zeros(2, dtype=torch.int64)), "keep"),
    (dict(weights=torch.zeros(2, 40)), "weights"),
])
def test_evict_refuses(change, word):
    import tabicl_mi355_paged as paged
    kp, vp = _pool()
    a = dict(weights=torch.zeros(2, 48), keep=4, recent=0)
    a.update(change)
    with pytest.raises(ValueError, match=word):
        paged.paged_evict(kp, vp, _table(), torch.zeros(2, dtype=torch.int32), a["weights"], a["keep"], a["recent"])


def test_abi_refuses_before_launch():
    import tabicl_mi355_native as nat
    lib = nat.load()
    a = 0x1000  # 16-byte aligned placeholder address: refused before any use

    def attn(D=64, R=64, H=8, Hq=8, pages=10, sp=None, dtype=0, q=a, scale=0.125, table=a, M=4, w=None, wsn=0, N=2, Tq=1,
             qs=(512, 64, 512), ws=a, wsb=1 << 40):
        return lib.tabicl_paged_attn(q, a, a, pages, H * R * D if sp is None else sp, R, table, M, M, a, w, wsn, a, N, Hq,
                                     H, Tq, D, *qs, 512, 64, 512, scale, dtype, ws, wsb, None)

    for kw, word in ((dict(D=48), "head dim"), (dict(R=24), "power of two"), (dict(R=8), "power of two"),
                     (dict(Hq=12), "multiple of H"), (dict(dtype=2), "dtype"), (dict(sp=512), "page stride"),
                     (dict(sp=8 * 64 * 64 + 4), "page stride"), (dict(q=a + 2), "aligned"), (dict(q=None), "aligned"),
                     (dict(scale=float("nan")), "scale"), (dict(table=None), "table"), (dict(M=1 << 30), "page counts"),
                     (dict(w=a, wsn=255), "weights"), (dict(qs=(512, 63, 512)), "strides"), (dict(N=70000), "65535"),
                     (dict(Tq=1 << 23), "query rows"), (dict(w=a, wsn=256, wsb=8), "workspace"),
                     (dict(pages=-1), "page counts"), (dict(w=a, wsn=1 << 30, M=1 << 20, N=9), "2^29"),
                     (dict(M=1 << 22, N=500), "2^37")):
        assert attn(**kw) == 1 and word in nat.last_error(), (kw, nat.last_error())
    assert attn(N=0) == 0 and attn(Tq=0, q=None) == 0
    assert lib.tabicl_paged_attn_workspace_bytes(2, 8, 8, 1, 48, 1000, 0, 0) < 0
    assert lib.tabicl_paged_attn_workspace_bytes(2, 8, 8, 1, 64, 1000, 1, 0) > 0
    assert lib.tabicl_paged_evict_workspace_bytes(-1, 4) < 0

    def append(T=3, k=a, ks=(64, 64, 64), N=2):
        return lib.tabicl_paged_append(a, a, 10, 8 * 64 * 64, 64, a, 4, 4, a, k, a, None, N, 8, T, 64, *ks, 64, 64, 64, 0,
                                       None)

    for kw, word in ((dict(T=-1), "row count"), (dict(k=a + 8), "aligned"), (dict(ks=(64, 64, 4)), "strides")):
        assert append(**kw) == 1 and word in nat.last_error(), (kw, nat.last_error())
    assert append(T=0) == 0 and append(N=0) == 0

    def gather(T=3, k=a, N=2, D=64):
        return lib.tabicl_paged_gather(a, a, 10, 8 * 64 * D, 64, a, 4, 4, a, k, a, N, 8, T, D, 0, None)

    for kw, word in ((dict(T=-1), "row count"), (dict(k=a + 4), "aligned"), (dict(k=None), "aligned"), (dict(D=48), "head dim")):
        assert gather(**kw) == 1 and word in nat.last_error(), (kw, nat.last_error())
    assert gather(T=0) == 0 and gather(N=0) == 0

    def evict(K=100, recent=0, ws=a, wsb=1 << 40, bsp=0, w=a, N=2, M=4):
        return lib.tabicl_paged_evict(a, a, 1, bsp, 10, 8 * 64 * 64, 64, a, M, M, a, w, 64 * M, None, 100, recent, a, K, a, a, N,
                                      8, 64, 0, ws, wsb, None)

    for kw, word in ((dict(K=257), "capacity"), (dict(recent=-1), "recent"), (dict(ws=None), "workspace"),
                     (dict(wsb=64), "workspace"), (dict(bsp=4), "block"), (dict(w=None), "weights"),
                     (dict(N=65000, M=1 << 10), "2^31")):
        assert evict(**kw) == 1 and word in nat.last_error(), (kw, nat.last_error())
    assert evict(N=0) == 0


def test_abi_evict_of_everything_needs_its_workspace():
    # K = 0 keeps nothing, but the number of moves still goes through the workspace
    import tabicl_mi355_native as nat
    a, need = 0x1000, nat.load().tabicl_paged_evict_workspace_bytes(2, 0)
    assert need > 0
    for ws, size in ((None, 1 << 40), (a, need - 1), (a + 8, need)):
        st = nat.load().tabicl_paged_evict(a, a, 1, 0, 10, 8 * 64 * 64, 64, a, 4, 4, a, a, 256, None, 0, 0, None, 0, a, a, 2, 8,
                                           64, 0, ws, size, None)
        assert st == 1 and "workspace" in nat.last_error()


# ---------------------------------------------------------------------------------------------
# PagedIclKVCache
# ---------------------------------------------------------------------------------------------
@pytest.fixture
def plain(monkeypatch):
    """The plain forms in place of the kernels."""
    import tabicl_mi355_native as nat
    import tabicl_mi355_paged as paged

    def attention(q, kp, vp, table, lengths, weights=None, scale=None, out=None):
        o, w, _, _ = ref.attention(q, kp, vp, table, lengths, q.shape[-1] ** -0.5 if scale is None else scale, weights)
        if weights is not None:
            weights.copy_(w)
        return o.to(q.dtype) if out is None else out.copy_(o)

    def append(kp, vp, table, lengths, k, v, count=None):
        a, b = ref.append(kp, vp, table, lengths, k, v, count)
        kp.copy_(a)
        vp.copy_(b)

    def evict(kp, vp, table, lengths, weights, keep, recent=0):
        a, b, *rest = ref.evict(kp, vp, table, lengths, weights, keep, recent)
        kp.copy_(a)
        vp.copy_(b)
        return tuple(rest)

    monkeypatch.setattr(nat, "require_device", lambda *t: None)
    for name, f in (("paged_attention", attention), ("paged_append", append), ("paged_evict", evict)):
        monkeypatch.setattr(paged, name, f)
    return paged


def _cache(paged, S=3, blocks=2, H=2, D=32, max_rows=100, pages=12, track=True):
    c = paged.PagedIclKVCache(S, blocks, H, D, max_rows, pages, 16, torch.float32, "cpu", track)
    c.keys.fill_(float("nan"))
    c.values.fill_(float("nan"))
    return c


def _rows(c, b, s):
    n = c.length(b, s)
    _, page, row = ref.rows_of(c.table[s], n, c.page_rows, c.keys.shape[1])
    return c.keys[b][page, :, row], c.values[b][page, :, row]


def test_cache_appends_and_queries(plain):
    g = torch.Generator().manual_seed(1)
    c = _cache(plain)
    assert c.shape == (3, 2, 2, 112, 32) and c.free_pages == 12
    want = {b: [(torch.zeros(0, 2, 32),) * 2 for _ in range(3)] for b in range(2)}
    with pytest.raises(ValueError, match="append before"):
        c.query(0, torch.zeros(3, 2, 1, 32))
    for rows in ([20, 1, 0], [1, 1, 1], [15, 40, 16], [0, 0, 0]):
        T = max(rows)
        for b in range(2):
            k, v = (torch.randn(3, 2, T, 32, generator=g) for _ in range(2))
            c.append(b, k, v, rows)
            for s in range(3):
                want[b][s] = tuple(torch.cat([o, x[s, :, :rows[s]].transpose(0, 1)]) for o, x in zip(want[b][s], (k, v)))
    for b in range(2):
        for s in range(3):
            for got, w in zip(_rows(c, b, s), want[b][s]):
                assert torch.equal(got, w)
        assert c.lengths[b].tolist() == [36, 42, 17] == [c.length(b, s) for s in range(3)]
    assert c.free_pages == 12 - 3 - 3 - 2
    assert (c.table >= 0).sum() == 8 and len(set(c.table[c.table >= 0].tolist())) == 8
    q = torch.randn(3, 2, 4, 32, generator=g)
    out = c.query(1, q)
    for s in range(3):
        k, v = want[1][s]
        p = torch.softmax(torch.einsum("htd,rhd->htr", q[s], k) * 32 ** -0.5, -1)
        assert torch.allclose(out[s], torch.einsum("htr,rhd->htd", p, v), atol=1e-5)
        assert torch.allclose(c.weights[s, :len(k)], p.sum((0, 1)), atol=1e-5)
    # a valid length, as a number and per sequence, and an output view
    for valid in (5, torch.tensor([5, 5, 5]), torch.tensor(5)):
        o = torch.zeros(3, 4, 2, 32)
        c.query(1, q, valid, out=o.transpose(1, 2))
        for s in range(3):
            k, v = want[1][s][0][:5], want[1][s][1][:5]
            p = torch.softmax(torch.einsum("htd,rhd->htr", q[s], k) * 32 ** -0.5, -1)
            assert torch.allclose(o[s], torch.einsum("htr,rhd->thd", p, v), atol=1e-5)
    view = c.estimators(1, 3)
    assert torch.allclose(view.query(1, q[1:]), out[1:], atol=1e-6)
    for b in range(2):  # the view shows what the cache gets later
        c.append(b, k[None].expand(3, -1, -1, -1).transpose(1, 2)[:, :, :5], v[None].expand(3, -1, -1, -1).transpose(1, 2)[:, :, :5])
    assert view.length(1, 0) == 47 and view.length(1, 1) == 22
    assert torch.allclose(view.estimators(1, 2).query(1, q[2:]), c.query(1, q)[2:], atol=1e-6)
    with pytest.raises(ValueError, match="queries only"):
        view.append(0, torch.zeros(2, 2, 1, 32), torch.zeros(2, 2, 1, 32))


def test_cache_evicts_and_reuses_pages(plain):
    g = torch.Generator().manual_seed(2)
    c = _cache(plain)
    k, v = (torch.randn(3, 2, 60, 32, generator=g) for _ in range(2))
    for b in range(2):
        c.append(b, k + b, v - b, [60, 33, 5])
    assert c.free_pages == 12 - 4 - 3 - 1
    c.query(0, torch.randn(3, 2, 3, 32, generator=g))
    before = c.weights.clone()
    index = c.evict(20, recent=2)
    assert index.shape == (3, 20) and c.free_pages == 12 - 2 - 2 - 1
    assert [c.length(1, s) for s in range(3)] == [20, 20, 5] and c.lengths.tolist() == [[20, 20, 5]] * 2
    for s, n in enumerate((20, 20, 5)):
        idx = index[s, :n].long()
        assert (index[s, n:] == -1).all() and len(set(idx.tolist())) == n
        for b in range(2):
            kb, vb = _rows(c, b, s)
            assert torch.equal(kb, (k[s] + b)[:, idx].transpose(0, 1)) and torch.equal(vb, (v[s] - b)[:, idx].transpose(0, 1))
        assert torch.equal(c.weights[s, :n], before[s, idx]) and (c.weights[s, n:] == 0).all()
    assert {58, 59} <= set(index[0].tolist())
    # the freed pages serve the next appends; a per-sequence budget; release
    for b in range(2):
        c.append(b, k[:, :, :30], v[:, :, :30], [30, 0, 30])
    assert c.free_pages == 12 - 4 - 2 - 3
    c.evict([50, 7, 0])
    assert [c.length(0, s) for s in range(3)] == [50, 7, 0] and c.free_pages == 12 - 4 - 1
    c.release(0)
    assert c.free_pages == 11 and c.length(0, 0) == 0 and (c.table[0] == -1).all() and (c.weights[0] == 0).all()


def test_cache_refuses(plain):
    c = _cache(plain, track=False)
    z = torch.zeros(3, 2, 4, 32)
    with pytest.raises(ValueError, match="power of two"):
        plain.PagedIclKVCache(1, 1, 2, 32, 100, 4, 24, device="cpu")
    with pytest.raises(ValueError, match="append expects"):
        c.append(0, z[:2], z[:2])
    with pytest.raises(ValueError, match="out of range"):
        c.append(2, z, z)
    with pytest.raises(ValueError, match="counts from 0"):
        c.append(0, z, z, [1, 2, 5])
    with pytest.raises(ValueError, match="cast"):
        c.append(0, z.bfloat16(), z.bfloat16())
    with pytest.raises(ValueError, match="capacity"):
        c.reserve(113)
    with pytest.raises(ValueError, match="pages wanted"):
        c.reserve(100)
    assert c.free_pages == 12 and (c.table == -1).all()  # a refused call changes nothing
    c.append(0, z, z)
    with pytest.raises(ValueError, match="track"):
        c.evict(2)
    with pytest.raises(ValueError, match="wider"):
        c.query(0, torch.zeros(3, 2, 1, 32, dtype=torch.float64))
    t = _cache(plain)
    t.append(0, z, z)
    with pytest.raises(ValueError, match="different rows"):
        t.evict(2)
    t.append(1, z, z)
    with pytest.raises(ValueError, match="keep"):
        t.evict([1, 2])
    with pytest.raises(ValueError, match="keep"):
        t.evict(-1)


def test_release_keeps_what_others_reserved(plain):
    c = _cache(plain)
    c.reserve([30, 50, 0])
    z = torch.zeros(3, 2, 10, 32)
    for b in range(2):
        c.append(b, z, z, [10, 3, 0])
    table = c.table.clone()
    assert c.free_pages == 12 - 2 - 4
    c.release(-3)
    assert c.free_pages == 12 - 4 and (c.table[0] == -1).all() and torch.equal(c.table[1], table[1])
    assert c.length(1, 1) == 3
    with pytest.raises(IndexError):
        c.release(3)
    c.release(1)
    assert c.free_pages == 12


@pytest.mark.parametrize("rows", [1, 2000])
def test_query_refuses_gradients(plain, rows):
    # at every number of query rows, also where the dense kernel would answer
    c = plain.PagedIclKVCache(1, 1, 1, 64, 64, 4, device="cpu")
    z = torch.zeros(1, 1, 8, 64, dtype=torch.bfloat16)
    c.append(0, z, z)
    q = torch.zeros(1, 1, rows, 64, dtype=torch.bfloat16, requires_grad=True)
    with pytest.raises(ValueError, match="no gradient"):
        c.query(0, q)
    with torch.no_grad():
        assert c.query(0, q).shape == q.shape


@pytest.mark.parametrize("N,H,G,D,rows,dtype", [
    (1, 8, 1, 64, 50048, 0), (8, 8, 1, 64, 8128, 0), (8, 8, 1, 64, 45056, 0), (8, 8, 1, 64, 45056, 1), (64, 8, 1, 64, 45056, 0),
    (64, 2, 12, 128, 1024, 1), (1, 8, 3, 32, 50048, 1), (3, 1, 64, 64, 21824, 0), (64, 8, 1, 64, 45056, 1)])
def test_workspace_is_bounded_in_the_query_rows(N, H, G, D, rows, dtype):
    # the scores kept for the weights: at most 1 GiB, or 16 query rows of every K/V head; 128 MiB cover the partials, the
    # references and the sums of up to 2^22 query rows
    import tabicl_mi355_native as nat
    scores = max(1 << 30, N * H * max(16, G) * rows * 4)
    sizes = [nat.load().tabicl_paged_attn_workspace_bytes(N, H * G, H, Tq, D, rows, 1, dtype)
             for Tq in (1, 8, 13, 64, 100, 1000, 5000, 20000) if N * H * G * Tq <= 1 << 22]
    assert all(0 < n <= scores + (128 << 20) for n in sizes), sizes


def test_query_rows_beyond_one_launch():
    # the query of 70,000 test rows by 8 estimators of 8 heads, which IclKVCache takes: slices, whatever the cache
    import tabicl_mi355_native as nat
    size = nat.load().tabicl_paged_attn_workspace_bytes
    for rows, weights, dtype in ((45056, 0, 0), (45056, 1, 0), (45056, 0, 1), (1024, 1, 0), (1 << 24, 0, 0)):
        assert 0 <= size(8, 8, 8, 70000, 64, rows, weights, dtype) <= (1152 << 20), (rows, weights, dtype, nat.last_error())
    assert size(8, 8, 8, 1 << 20, 64, 45056, 0, 0) > 0
    for n in ((8, 8, 8, (1 << 20) + 1, 64, 45056, 0, 0), (1, 1, 1, (1 << 22) + 1, 64, 64, 0, 0), (65535, 128, 1, 1, 64, 64, 0, 0)):
        assert size(*n) < 0 and "query rows" in nat.last_error()


def test_gather_of_ragged_tables_is_bounded(plain, monkeypatch):
    # one long table among short ones: K and V side by side never take more than the bound, except a single table's own
    lengths = [3, 0, 900, 20, 1, 300, 300, 300, 7]
    c = plain.PagedIclKVCache(9, 1, 2, 64, 1000, 150, 16, torch.bfloat16, "cpu")
    g = torch.Generator().manual_seed(5)
    k, v = (torch.randn(9, 2, 900, 64, generator=g).bfloat16() for _ in range(2))
    c.append(0, k, v, lengths)
    row, taken = 2 * 2 * 64 * 2, []

    def gather(kp, vp, table, n, rows):
        taken.append((table.shape[0], table.shape[0] * rows * row))
        out = [torch.full((table.shape[0], 2, rows, 64), float("nan"), dtype=torch.bfloat16) for _ in range(2)]
        for s in range(table.shape[0]):
            at, page, r = ref.rows_of(table[s], min(int(n[s]), rows), 16, kp.shape[0])
            for o, pages in zip(out, (kp, vp)):
                o[s][:, at] = pages[page, :, r].transpose(0, 1)
        return out

    def dense(q, kd, vd, n, out):
        o = torch.zeros(q.shape, dtype=q.dtype)
        for s in range(len(n)):
            m = int(n[s])
            if m:
                p = torch.softmax(q[s].double() @ kd[s, :, :m].double().transpose(1, 2) / 8, -1)
                o[s] = (p @ vd[s, :, :m].double()).to(q.dtype)
        return o if out is None else out.copy_(o)

    monkeypatch.setattr(plain, "paged_gather", gather)
    monkeypatch.setattr(plain.PagedIclKVCache, "_dense", staticmethod(dense))
    monkeypatch.setattr(plain, "_DENSE_SCORES", 1)
    monkeypatch.setattr(plain, "_GATHER_BYTES", 700 * row, raising=False)
    q = torch.randn(9, 300, 2, 64, generator=g).bfloat16().transpose(1, 2)
    for valid in (None, 250, torch.tensor([900, 9, 700, 2, 2, 2, 300, 300, 300])):
        taken.clear()
        want = [min(n, 900 if valid is None else int(valid) if not torch.is_tensor(valid) else int(valid[s])) for s, n in
                enumerate(lengths)]
        buf = torch.zeros(9, 300, 2, 64, dtype=torch.bfloat16)
        got = c.query(0, q, valid)
        assert c.query(0, q, valid, buf.transpose(1, 2)).data_ptr() == buf.data_ptr()
        assert torch.equal(got, buf.transpose(1, 2))
        assert all(size <= 700 * row or n == 1 for n, size in taken), taken
        for s, n in enumerate(want):
            assert torch.equal(got[s], dense(q[s:s + 1], k[s:s + 1], v[s:s + 1], [n], None)[0]), (valid, s)


@pytest.mark.parametrize("T", [1, 600])
def test_query_shapes(plain, monkeypatch, T):
    # the same heads at every number of query rows: groups of them too, and a refusal that names what is expected
    monkeypatch.setattr(plain, "_DENSE_SCORES", 1)
    c = plain.PagedIclKVCache(2, 1, 2, 64, 64, 8, 16, torch.bfloat16, "cpu")
    g = torch.Generator().manual_seed(6)
    k, v = (torch.randn(2, 2, 40, 64, generator=g).bfloat16() for _ in range(2))
    c.append(0, k, v, [40, 7])
    q = torch.randn(2, 6, T, 64, generator=g).bfloat16()
    got = c.query(0, q)
    for s, n in enumerate((40, 7)):
        for h in range(6):
            p = torch.softmax(q[s, h].double() @ k[s, h // 3, :n].double().t() / 8, -1)
            assert torch.equal(got[s, h], (p @ v[s, h // 3, :n].double()).to(q.dtype))
    for shape in ((3, 2, T, 64), (1, 2, T, 64), (2, 3, T, 64), (2, 0, T, 64), (2, 1, T, 64), (2, 2, T, 32), (2, 2, 64), (T, 64)):
        with pytest.raises(ValueError, match="query expects"):
            c.query(0, torch.zeros(shape, dtype=torch.bfloat16))


def test_chunks_of_empty_tables(plain):
    # a chunk without a row answers as the whole query does: 0
    c = _cache(plain)
    g = torch.Generator().manual_seed(7)
    k, v = (torch.randn(3, 2, 20, 32, generator=g) for _ in range(2))
    for b in range(2):
        c.append(b, k, v, [20, 0, 5])
    c.release(2)
    q = torch.randn(3, 2, 4, 32, generator=g)
    want = c.query(1, q)
    assert (want[1:] == 0).all() and (want[0] != 0).any()
    for a, b in ((0, 1), (1, 2), (2, 3), (1, 3)):
        assert torch.equal(c.estimators(a, b).query(1, q[a:b]), want[a:b])
    views = [c.estimators(s, s + 1) for s in range(3)]
    c.release(0)  # nothing left: refused, by the cache and by its views
    for x, y in [(c, q)] + [(w, q[:1]) for w in views]:
        with pytest.raises(ValueError, match="append before"):
            x.query(1, y)


def test_valid_lengths_of_other_types(plain):
    # numbers beyond 32 bits mean no limit, as a tensor too
    c = _cache(plain)
    g = torch.Generator().manual_seed(8)
    k, v = (torch.randn(3, 2, 20, 32, generator=g) for _ in range(2))
    c.append(1, k, v, [20, 3, 5])
    q = torch.randn(3, 2, 4, 32, generator=g)
    free, cut = c.query(1, q), c.query(1, q, torch.tensor([4, 4, 4], dtype=torch.int32))
    for big in (2 ** 63 - 1, 2 ** 31, 2 ** 32 + 4):
        for valid in (big, torch.tensor(big), torch.tensor([big]), torch.tensor([big, 2 ** 40, 20])):
            assert torch.equal(c.query(1, q, valid), free), valid
    for valid in (4, torch.tensor([4]), torch.tensor([4, 4, 4]), torch.tensor([4, 2 ** 40, 4]).clamp(max=4),
                  torch.tensor([4] * 3, dtype=torch.uint8), torch.tensor([4] * 3, dtype=torch.int16)):
        assert torch.equal(c.query(1, q, valid), cut), valid
    for none in (0, -1, torch.tensor(-2 ** 40), torch.tensor([0, -1, -2 ** 63])):
        assert (c.query(1, q, none) == 0).all(), none


def test_forward_tangents_are_refused():
    # as gradients in reverse mode are: none of the operators carries a tangent on
    import torch.autograd.forward_ad as fw
    import tabicl_mi355_native as nat
    import tabicl_mi355_paged as paged
    k, v = _pool()
    t, n, q, w = _table(), torch.tensor([5, 9], dtype=torch.int32), torch.zeros(2, 2, 1, 64), torch.zeros(2, 48)
    calls = {"q": lambda x: paged.paged_attention(x, k, v, t, n), "k_pages": lambda x: paged.paged_attention(q, x, v, t, n),
             "v_pages": lambda x: paged.paged_attention(q, k, x, t, n), "weights": lambda x: paged.paged_attention(q, k, v, t, n, x),
             "out": lambda x: paged.paged_attention(q, k, v, t, n, None, None, x), "k": lambda x: paged.paged_append(k, v, t, n, x, q),
             "v": lambda x: paged.paged_append(k, v, t, n, q, x), "append": lambda x: paged.paged_append(x, v, t, n, q, q),
             "gather": lambda x: paged.paged_gather(k, x, t, n, 3), "evict": lambda x: paged.paged_evict(x, v, t, n, w, 3),
             "evict weights": lambda x: paged.paged_evict(k, v, t, n, x, 3)}
    args = dict.fromkeys(("q", "out", "k", "v"), q) | dict.fromkeys(("weights", "evict weights"), w)
    for name, call in calls.items():
        x = args.get(name, k)
        with fw.dual_level():
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(ValueError, match="no gradient"):
                    call(fw.make_dual(x.clone(), torch.ones_like(x)))
            with pytest.raises(nat.NativeLibraryError):  # a level alone changes nothing
                call(x)
        with pytest.raises(ValueError, match="no gradient"):
            torch.func.jvp(call, (x.clone(),), (torch.ones_like(x),))


def test_query_refuses_forward_tangents(plain):
    import torch.autograd.forward_ad as fw
    c = plain.PagedIclKVCache(1, 1, 1, 64, 64, 4, 16, torch.float32, "cpu")
    z = torch.zeros(1, 1, 8, 64)
    c.append(0, z, z)
    with fw.dual_level():
        for T in (2, 2000):
            q = torch.zeros(1, 1, T, 64)
            with torch.no_grad(), pytest.raises(ValueError, match="no gradient"):
                c.query(0, fw.make_dual(q, torch.ones_like(q)))
            assert c.query(0, q).shape == q.shape


def test_workspace_sizes_do_not_pile_up(monkeypatch):
    # what is kept of workspace sizes has a bound, for evictions (whose sizes change with the data) as for queries
    import tabicl_mi355_native as nat
    import tabicl_mi355_paged as paged
    monkeypatch.setattr(paged, "_WS_BYTES", {})
    k, v = _pool()
    t, n = _table(), torch.tensor([5, 9], dtype=torch.int32)
    table = torch.zeros(2, 400, dtype=torch.int32)
    monkeypatch.setattr(nat, "call", lambda *a: None)
    monkeypatch.setattr(nat, "require_device", lambda *a: None)
    monkeypatch.setattr(nat, "stream_of", lambda *a: 0)
    monkeypatch.setattr(nat, "direct", lambda *a: True)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda self: 0)
    w = torch.zeros(2, 6400)
    for keep in range(5000):
        paged.paged_evict(k, v, table, n, w, keep)
        assert len(paged._WS_BYTES) <= 4096
    for width in range(1, 400, 7):
        for T in range(1, 90):
            paged.paged_attention(torch.zeros(2, 2, T, 64), k, v, table[:, :width], n)
        assert len(paged._WS_BYTES) <= 4096


def test_refused_append_takes_no_pages(plain):
    c = _cache(plain)
    k = torch.zeros(3, 2, 20, 32, requires_grad=True)
    z = torch.zeros(3, 2, 20, 32)
    for a, b in ((k, z), (z, k)):
        with pytest.raises(ValueError, match="no gradient"):
            c.append(0, a, b)
    assert c.free_pages == 12 and (c.table == -1).all() and c.length(0, 0) == 0
    with torch.no_grad():
        c.append(0, k, k)
    assert c.length(0, 2) == 20


@pytest.mark.parametrize("inside", [True, False])
def test_cache_built_in_inference_mode(plain, inside):
    # built by a service's set-up in inference mode, filled and asked in or outside of it, as IclKVCache can be
    with torch.inference_mode():
        c = plain.PagedIclKVCache(2, 1, 2, 32, 60, 8, 16, torch.float32, "cpu", track=True)
    g = torch.Generator().manual_seed(9)
    with torch.inference_mode(inside):
        k, v, q = (torch.randn(2, 2, 20, 32, generator=g) for _ in range(3))
        c.append(0, k, v, [20, 4])
        c.query(0, q)
        c.evict(10)
        c.release(1)
        c.append(0, k, v)
    assert c.lengths.tolist() == [[30, 20]] and c.free_pages == 8 - 2 - 2


def test_chunks_with_a_valid_length_per_table(plain):
    # one length per table goes to the chunks table by table, as one for all does
    import tabicl_mi355_icl as icl
    g = torch.Generator().manual_seed(10)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    blocks = [icl.IclBlockWeights(r(64), r(64), r(192, 64) / 8, None, r(64, 64) / 8, None, r(64), r(64), r(128, 64) / 8, None,
                                  r(64, 128) / 11, None) for _ in range(2)]
    c = _cache(plain, track=False)
    for b in range(2):
        c.append(b, r(3, 2, 20, 32), r(3, 2, 20, 32), [20, 11, 4])
    x = r(3, 5, 64)
    for valid in (None, 6, torch.tensor(6), torch.tensor([6]), torch.tensor([9, 2, 20]), torch.tensor([[9], [2], [20]])):
        with torch.no_grad():
            want = c.query_blocks(x, blocks, valid)
            for chunks in ([(0, 3)], [(0, 1), (1, 3)], [(0, 1), (1, 2), (2, 3)]):
                assert torch.allclose(c.query_chunked(x, blocks, chunks, valid), want, atol=1e-5), (valid, chunks)


@pytest.mark.parametrize("S,T,gathered", [(1, 384, False), (1, 1023, False), (1, 1024, True), (2, 500, False), (2, 512, True),
                                          (8, 128, False), (4, 256, True)])
def test_few_query_rows_over_all_tables_stay_in_the_pages(plain, monkeypatch, S, T, gathered):
    monkeypatch.setattr(plain, "_DENSE_SCORES", 1)
    c = plain.PagedIclKVCache(S, 1, 1, 64, 16, S, 16, torch.bfloat16, "cpu")
    z = torch.zeros(S, 1, 4, 64, dtype=torch.bfloat16)
    c.append(0, z, z)
    calls = []
    monkeypatch.setattr(plain, "paged_gather", lambda kp, vp, table, n, rows: calls.append(rows) or (z[:, :, :rows],) * 2)
    monkeypatch.setattr(plain.PagedIclKVCache, "_dense", staticmethod(lambda q, k, v, n, out: torch.zeros_like(q)))
    q = torch.zeros(S, 1, T, 64, dtype=torch.bfloat16)
    assert c.query(0, q).shape == q.shape and calls == [4] * gathered
