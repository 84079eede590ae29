"""CPU tests of the 8-bit paged cache, of attention over selected pages and of the books on the GPU: what the wrappers and the C
ABI refuse, and PagedIclKVCache's use of them with the plain forms in the kernels' place."""
import pytest
import torch

import paged8_ref as ref
import paged_ref

BF, F32, E4, I8, I32 = torch.bfloat16, torch.float32, torch.float8_e4m3fn, torch.int8, torch.int32


def _args(**change):
    a = dict(q=torch.zeros(2, 2, 1, 64), k=torch.zeros(6, 2, 16, 64).to(E4), v=torch.zeros(6, 2, 16, 64).to(E4),
             table=torch.arange(6, dtype=I32).view(2, 3), lengths=torch.tensor([5, 9], dtype=I32), scales=torch.ones(6, 2, 2),
             rows=torch.zeros(2, 2, 4, 64), rows_v=None, count=None, weights=None, out=None, bounds=torch.zeros(6, 2, 2, 64, dtype=I8),
             bound_scales=torch.ones(6, 2), index=torch.zeros(2, 2, 1, 3, dtype=I32), start=None)
    assert not set(change) - set(a)
    a.update(change)
    return a


def test_no_cpu_path():
    import tabicl_mi355_native as nat
    import tabicl_mi355_paged as paged
    a = _args()
    p = (a["k"], a["v"], a["table"], a["lengths"])
    count, free, fc = torch.ones(2, dtype=I32), torch.zeros(6, dtype=I32), torch.zeros(1, dtype=I32)
    for call in (lambda: paged.paged_attention(a["q"], *p, scales=a["scales"]),
                 lambda: paged.paged_append(*p, a["rows"], a["rows"], scales=a["scales"]),
                 lambda: paged.paged_gather(*p, 4, scales=a["scales"]),
                 lambda: paged.paged_bounds(a["k"], a["table"], a["lengths"], a["bounds"], a["bound_scales"], scales=a["scales"]),
                 lambda: paged.paged_select(a["q"], a["bounds"], a["bound_scales"], a["table"], a["lengths"], 16, 2),
                 lambda: paged.paged_sparse_attention(a["q"], *p, a["index"], scales=a["scales"]),
                 lambda: paged.paged_reserve(a["table"], a["lengths"], count, free, fc, 16),
                 lambda: paged.paged_release(a["table"], a["lengths"], free, fc, 16),
                 lambda: paged.paged_slots(a["table"], a["lengths"], count, 2, 6, 16),
                 lambda: paged.paged_append_packed(a["k"].float(), a["v"].float(), a["table"], a["lengths"], count, torch.zeros(2, 2, 64),
                                                   torch.zeros(2, 2, 64), torch.zeros(2, dtype=torch.int64), torch.zeros(3, dtype=I32)),
                 lambda: paged.paged_append_packed(*p, count, torch.zeros(2, 2, 64), torch.zeros(2, 2, 64),
                                                   torch.zeros(2, dtype=torch.int64), torch.zeros(3, dtype=I32), a["scales"])):
        with pytest.raises(nat.NativeLibraryError):
            call()


@pytest.mark.parametrize("change,word", [
    (dict(q=torch.zeros(2, 3, 1, 64)), "multiple of 2 heads"),
    (dict(q=torch.zeros(2, 2, 1, 32)), "must be"),
    (dict(q=torch.zeros(2, 2, 1, 64, dtype=torch.float16)), "not supported"),
    (dict(scales=None), "needs its scales"),
    (dict(scales=torch.ones(6, 2)), "scales must be"),
    (dict(scales=torch.ones(6, 2, 2, dtype=torch.float64)), "scales must be"),
    (dict(scales=torch.ones(2, 6, 2).transpose(0, 1)), "scales must be"),
    (dict(scales=torch.ones(25)[1:].view(6, 2, 2)), "scales must be"),
    (dict(k=torch.zeros(6, 2, 16, 64, dtype=I8)), "share a dtype"),
    (dict(k=torch.zeros(6, 2, 16, 64), v=torch.zeros(6, 2, 16, 64)), "8-bit codes"),
    (dict(weights=torch.zeros(2, 48)), "no weights"),
    (dict(out=torch.zeros(2, 2, 2, 64)), "out"),
    (dict(out=torch.zeros(2, 2, 1, 64, dtype=BF)), "out"),
    (dict(table=torch.zeros(2, 3, dtype=torch.int64)), "int32"),
    (dict(lengths=torch.zeros(3, dtype=I32)), "lengths"),
    (dict(q=torch.zeros(2, 2, 1, 64, requires_grad=True)), "no gradient"),
])
def test_attention_refuses(change, word):
    import tabicl_mi355_paged as paged
    a = _args(**change)
    with pytest.raises(ValueError, match=word):
        paged.paged_attention(a["q"], a["k"], a["v"], a["table"], a["lengths"], a["weights"], None, a["out"], a["scales"])


@pytest.mark.parametrize("change,word", [
    (dict(rows=torch.zeros(2, 2, 4, 32)), "must be"),
    (dict(rows=torch.zeros(2, 2, 64)), "must be"),
    (dict(rows_v=torch.zeros(2, 2, 3, 64)), "must be"),
    (dict(rows_v=torch.zeros(2, 2, 4, 64, dtype=BF)), "share a dtype"),
    (dict(rows=torch.zeros(2, 2, 4, 64, dtype=torch.float16)), "not supported"),
    (dict(count=torch.zeros(2, dtype=torch.int64)), "count"),
    (dict(scales=None), "needs its scales"),
    (dict(rows=torch.zeros(2, 2, 4, 64, requires_grad=True)), "no gradient"),
])
def test_append_refuses(change, word):
    import tabicl_mi355_paged as paged
    a = _args(**change)
    with pytest.raises(ValueError, match=word):
        paged.paged_append(a["k"], a["v"], a["table"], a["lengths"], a["rows"], a["rows"] if a["rows_v"] is None else a["rows_v"],
                           a["count"], a["scales"])


def test_gather_refuses():
    import tabicl_mi355_paged as paged
    a = _args()
    p = (a["k"], a["v"], a["table"], a["lengths"])
    for call in (lambda: paged.paged_gather(*p, 4), lambda: paged.paged_gather(*p, -1, scales=a["scales"]),
                 lambda: paged.paged_gather(*p, 4, a["scales"], torch.float16),
                 lambda: paged.paged_gather(a["k"].float(), a["v"].float(), *p[2:], 4, dtype=BF),
                 lambda: paged.paged_gather(a["k"].float(), a["v"].float(), *p[2:], 4, a["scales"])):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("change,word", [
    (dict(bounds=torch.zeros(6, 2, 2, 32, dtype=I8)), "bounds must"),
    (dict(bounds=torch.zeros(6, 2, 2, 64)), "bounds must"),
    (dict(bounds=torch.zeros(6, 2, 64, 2, dtype=I8).transpose(2, 3)), "bounds must"),
    (dict(bound_scales=torch.ones(6, 3)), "bound_scales must"),
    (dict(start=torch.zeros(2)), "start"),
    (dict(scales=None), "needs its scales"),
    (dict(bound_scales=torch.ones(6, 2, requires_grad=True)), "no gradient"),
])
def test_bounds_refuse(change, word):
    import tabicl_mi355_paged as paged
    a = _args(**change)
    with pytest.raises(ValueError, match=word):
        paged.paged_bounds(a["k"], a["table"], a["lengths"], a["bounds"], a["bound_scales"], a["start"], None, a["scales"])
    with pytest.raises(ValueError, match="negative"):
        paged.paged_bounds(a["k"], a["table"], a["lengths"], a["bounds"], a["bound_scales"], None, -1, a["scales"])


@pytest.mark.parametrize("change,word", [
    (dict(q=torch.zeros(2, 3, 1, 64)), "multiple of 2 heads"),
    (dict(q=torch.zeros(2, 2, 64)), "paged_select needs"),
    (dict(bounds=torch.zeros(6, 2, 128, dtype=I8)), "paged_select needs"),
    (dict(bound_scales=torch.ones(6)), "bound_scales"),
    (dict(table=torch.zeros(2, 3)), "int32"),
    (dict(q=torch.zeros(2, 2, 1, 64, requires_grad=True)), "no gradient"),
])
def test_select_refuses(change, word):
    import tabicl_mi355_paged as paged
    a = _args(**change)
    with pytest.raises(ValueError, match=word):
        paged.paged_select(a["q"], a["bounds"], a["bound_scales"], a["table"], a["lengths"], 16, 2)
    with pytest.raises(ValueError, match="negative"):
        paged.paged_select(a["q"], a["bounds"], a["bound_scales"], a["table"], a["lengths"], 16, -2)


@pytest.mark.parametrize("change,word", [
    (dict(index=torch.zeros(2, 2, 1, 3)), "index must"),
    (dict(index=torch.zeros(2, 1, 1, 3, dtype=I32)), "index must"),
    (dict(index=torch.zeros(2, 2, 3, 1, dtype=I32).transpose(2, 3).expand(2, 2, 1, 3)[..., ::2]), "index must"),
    (dict(q=torch.zeros(2, 2, 1, 32)), "must be"),
    (dict(k=torch.zeros(6, 2, 16, 64).to(BF), v=torch.zeros(6, 2, 16, 64).to(BF), scales=None), "cast q"),
    (dict(k=torch.zeros(6, 2, 16, 64), v=torch.zeros(6, 2, 16, 64)), "8-bit codes"),
    (dict(scales=None), "needs its scales"),
    (dict(out=torch.zeros(2, 2, 1, 1).expand(2, 2, 1, 64)), "out"),
    (dict(q=torch.zeros(2, 2, 1, 64, requires_grad=True)), "no gradient"),
])
def test_sparse_attention_refuses(change, word):
    import tabicl_mi355_paged as paged
    a = _args(**change)
    with pytest.raises(ValueError, match=word):
        paged.paged_sparse_attention(a["q"], a["k"], a["v"], a["table"], a["lengths"], a["index"], None, a["out"], a["scales"])


def test_books_refuse():
    import tabicl_mi355_paged as paged
    t, n, c = torch.zeros(2, 3, dtype=I32), torch.zeros(2, dtype=I32), torch.ones(2, dtype=I32)
    f, fc = torch.zeros(6, dtype=I32), torch.zeros(1, dtype=I32)
    for call, word in (
            (lambda: paged.paged_reserve(t.long(), n, c, f, fc, 16), "table"),
            (lambda: paged.paged_reserve(t, n.long(), c, f, fc, 16), "lengths"),
            (lambda: paged.paged_reserve(t, n, c[:1], f, fc, 16), "count"),
            (lambda: paged.paged_reserve(t, n, c, f.long(), fc, 16), "free must"),
            (lambda: paged.paged_reserve(t, n, c, f.view(2, 3), fc, 16), "free must"),
            (lambda: paged.paged_reserve(t, n, c, f, fc.long(), 16), "free_count"),
            (lambda: paged.paged_release(t, n, f, f, 16), "free_count"),
            (lambda: paged.paged_release(t.t(), n, f, fc, 16), "table"),
            (lambda: paged.paged_reserve(t[:1].expand(2, 3), n, c, f, fc, 16), "overlap"),
            (lambda: paged.paged_release(torch.zeros(5, dtype=I32).as_strided((2, 3), (2, 1)), n, f, fc, 16), "overlap"),
            (lambda: paged.paged_slots(t, n, c, -1, 6, 16), "negative"),
            (lambda: paged.paged_slots(t, n, c.float(), 2, 6, 16), "count"),
            (lambda: paged.paged_append_packed(torch.zeros(6, 2, 16, 64), torch.zeros(6, 2, 16, 64), t, n, c, torch.zeros(2, 2, 32),
                                               torch.zeros(2, 2, 32), torch.zeros(2, dtype=torch.int64), torch.zeros(3, dtype=I32)), "k and v"),
            (lambda: paged.paged_append_packed(torch.zeros(6, 2, 16, 64), torch.zeros(6, 2, 16, 64), t, n, c, torch.zeros(2, 2, 64),
                                               torch.zeros(2, 2, 64), torch.zeros(2, dtype=I32), torch.zeros(3, dtype=I32)), "slots"),
            (lambda: paged.paged_append_packed(torch.zeros(6, 2, 16, 64).to(E4), torch.zeros(6, 2, 16, 64).to(E4), t, n, c,
                                               torch.zeros(2, 2, 64), torch.zeros(2, 2, 64), torch.zeros(2, dtype=torch.int64),
                                               torch.zeros(2, dtype=I32), torch.ones(6, 2, 2)), "starts")):
        with pytest.raises(ValueError, match=word):
            call()


def test_abi_refuses_before_launch():
    import tabicl_mi355_native as nat
    lib = nat.load()
    a = 0x1000  # 16-byte aligned placeholder address: refused before any use

    def attn(D=64, R=64, H=8, Hq=8, pages=10, sp=None, dtype=0, code=0, q=a, scale=0.125, M=4, N=2, Tq=1, qs=512, sc=a, ws=a,
             wsb=1 << 40):
        return lib.tabicl_paged_attn_q8(q, a, a, sc, pages, H * R * D if sp is None else sp, R, a, M, M, a, a, N, Hq, H, Tq, D, qs, 64,
                                        512, 512, 64, 512, scale, dtype, code, ws, wsb, None)

    for kw, word in ((dict(D=48), "head dim"), (dict(R=24), "power of two"), (dict(Hq=12), "multiple of H"), (dict(dtype=2), "dtype"),
                     (dict(code=2), "code"), (dict(sc=None), "scales"), (dict(sc=a + 4), "scales"), (dict(sp=512), "page stride"),
                     (dict(sp=8 * 64 * 64 + 8), "page stride"), (dict(q=a + 2), "aligned"), (dict(scale=float("inf")), "scale"),
                     (dict(qs=513), "strides"), (dict(N=70000), "65535"), (dict(M=100, wsb=8), "workspace")):
        assert attn(**kw) == 1 and word in nat.last_error(), (kw, nat.last_error())
    assert attn(N=0) == 0 and attn(Tq=0, q=None) == 0

    def append(T=4, code=0, k=a, starts=None, count=None, ks=64, M=4, R=64, N=2):
        return lib.tabicl_paged_append_q8(a, a, a, 10, 8 * R * 64, R, a, M, M, a, k, a, count, starts, N, 8, T, 64, 512, 64, ks, 512, 64,
                                          512, 0, code, None)

    for kw, word in ((dict(T=-1), "row count"), (dict(code=7), "code"), (dict(k=a + 8), "aligned"), (dict(starts=a), "count"),
                     (dict(ks=60), "strides"), (dict(M=1 << 24, T=1 << 30), "2^22")):
        assert append(**kw) == 1 and word in nat.last_error(), (kw, nat.last_error())
    assert append(T=0) == 0 and append(N=0) == 0
    assert lib.tabicl_paged_gather_q8(a, a, a, 10, 8 * 64 * 64, 64, a, 4, 4, a, a + 8, a, 2, 8, 4, 64, 0, 0, None) == 1
    assert "aligned" in nat.last_error()

    def bounds(fmt=0, sc=None, bnd=a, rows=10, M=4, R=64):
        return lib.tabicl_paged_bounds(a, sc, 10, 8 * R * 64, R, a, M, M, a, a, rows, bnd, a, 2, 8, 64, fmt, None)

    for kw, word in ((dict(fmt=4), "format"), (dict(fmt=2), "scales"), (dict(bnd=a + 8), "bounds"), (dict(rows=-1), "negative"),
                     (dict(rows=1 << 30, M=1 << 24, R=16), "2^25")):
        assert bounds(**kw) == 1 and word in nat.last_error(), (kw, nat.last_error())

    def select(K=3, q=a, index=a, M=4, Tq=1, ws=None, wsb=0, N=2, dtype=0):
        return lib.tabicl_paged_select(q, a, a, 10, 16, a, M, M, a, index, K, N, 8, 8, Tq, 64, 512, 64, 512, dtype, ws, wsb, None)

    for kw, word in ((dict(K=-1), "page count"), (dict(q=a + 4), "aligned"), (dict(index=None), "index"), (dict(dtype=3), "dtype"),
                     (dict(Tq=1 << 18), "2^21"), (dict(M=40000), "workspace")):
        assert select(**kw) == 1 and word in nat.last_error(), (kw, nat.last_error())
    assert select(K=0) == 0 and select(N=0) == 0
    assert lib.tabicl_paged_select_workspace_bytes(2, 8, 1, 32768) == 0 < lib.tabicl_paged_select_workspace_bytes(2, 8, 1, 32769)
    assert lib.tabicl_paged_select_workspace_bytes(2, 8, -1, 10) < 0

    def sparse(fmt=0, dtype=0, K=3, index=a, ws=a, wsb=1 << 40, sc=None, Tq=1, N=2):
        return lib.tabicl_paged_sparse_attn(a, a, a, sc, 10, 8 * 64 * 64, 64, a, 4, 4, a, index, K, a, N, 8, 8, Tq, 64, 512, 64, 512, 512,
                                            64, 512, 0.1, dtype, fmt, ws, wsb, None)

    for kw, word in ((dict(fmt=1), "own dtype"), (dict(fmt=3), "scales"), (dict(fmt=9), "format"), (dict(dtype=2), "dtype"),
                     (dict(K=1 << 30), "page count"), (dict(index=None), "index"), (dict(K=64, wsb=16), "workspace"),
                     (dict(Tq=1 << 20), "2^22")):
        assert sparse(**kw) == 1 and word in nat.last_error(), (kw, nat.last_error())
    assert sparse(N=0) == 0

    for kw, word in ((dict(R=20), "power of two"), (dict(N=70000), "65535"), (dict(M=-1), "page counts"), (dict(c=None), "count"),
                     (dict(ws=None), "workspace")):
        p = dict(R=16, N=2, M=4, c=a, ws=a)
        p.update(kw)
        assert lib.tabicl_paged_reserve(a, 4, p["M"], a, p["c"], a, a, a, 10, p["R"], p["N"], p["ws"], 1 << 20, None) == 1
        assert word in nat.last_error(), (kw, nat.last_error())
    assert lib.tabicl_paged_reserve(a, 4, 4, a, a, a, a, a, 10, 16, 0, None, 0, None) == 0
    assert lib.tabicl_paged_release(a, 4, 4, a, None, a, 10, 16, 2, a, 1 << 20, None) == 1
    assert lib.tabicl_paged_slots(a, 4, 4, a, a, None, a, 5, 10, 16, 2, None) == 1
    assert lib.tabicl_paged_slots(a, 4, 4, a, a, a, a, 1 << 31, 10, 16, 2, None) == 1 and "total" in nat.last_error()
    assert lib.tabicl_paged_append_slots(a, a, 10, 8 * 16 * 64, 16, None, a, a, 4, 8, 64, 512, 64, 512, 64, 0, None) == 1
    assert lib.tabicl_paged_append_slots(a, a, 10, 8 * 16 * 64, 16, a, a, a, 4, 8, 64, 511, 64, 512, 64, 0, None) == 1
    assert "strides" in nat.last_error()
    assert lib.tabicl_paged_books_workspace_bytes(-1) < 0 < lib.tabicl_paged_books_workspace_bytes(0)


# ---------------------------------------------------------------------------------------------
# the plain forms themselves, and PagedIclKVCache with them
# ---------------------------------------------------------------------------------------------
def test_codes_are_those_of_torch():
    x = torch.cat([torch.linspace(-470, 470, 9001), torch.randn(5000) * 0.01, torch.tensor([0.0, -0.0, 2.0 ** -10, 3 * 2.0 ** -10])])
    assert torch.equal(ref.codes(x.double(), E4), x.clamp(-448, 448).to(E4).double())
    assert torch.equal(ref.codes(x.double(), I8), x.clamp(-127, 127).round().double())
    for top in (448.0, 127.0):
        for m in (0.0, 1e-30, top, top * (1 + 1e-9), 1.0, 3e38, float(top) / 8):
            k = ref.exponent(m, top)
            assert -60 <= k <= 100 and (m <= top * 2.0 ** k or k == 100) and (k == -60 or m > top * 2.0 ** (k - 1))


@pytest.fixture
def plain(monkeypatch):
    """The plain forms in place of the kernels."""
    import tabicl_mi355_native as nat
    import tabicl_mi355_paged as paged

    def values(pages, scales, which):
        return pages.double() if scales is None else ref.values(pages, scales, which)

    def attention(q, kp, vp, table, lengths, weights=None, scale=None, out=None, scales=None):
        o, _, _, _ = paged_ref.attention(q, values(kp, scales, 0), values(vp, scales, 1), table, lengths, q.shape[-1] ** -0.5)
        return o.to(q.dtype) if out is None else out.copy_(o)

    def append(kp, vp, table, lengths, k, v, count=None, scales=None, starts=None):
        a, b, s = ref.append(kp, vp, scales, table, lengths, k, v, count, starts)
        for to, x in ((kp, a), (vp, b), (scales, s)):
            to.copy_(x.to(to.dtype))

    def packed(kp, vp, table, lengths, count, k, v, slots, starts, scales=None):
        append(kp, vp, table, lengths, k, v, count, scales, starts)

    def slots(table, lengths, count, total, pages, R):
        s, st = ref.Books(table.tolist(), [], 0, pages, R).slots(lengths.tolist(), count.tolist(), total)
        return torch.tensor(s), torch.tensor(st, dtype=I32)

    def bounds(kp, table, lengths, bnd, bs, start=None, rows=None, scales=None):
        for (page, h), (hi, lo, step) in ref.bounds(values(kp, scales, 0), table, lengths, start).items():
            bnd[page, h, 0], bnd[page, h, 1], bs[page, h] = hi.to(I8), lo.to(I8), step

    def sparse(q, kp, vp, table, lengths, index, scale=None, out=None, scales=None):
        o, _ = ref.sparse_attention(q, values(kp, scales, 0), values(vp, scales, 1), table, lengths, index, q.shape[-1] ** -0.5)
        return o.to(q.dtype) if out is None else out.copy_(o)

    monkeypatch.setattr(nat, "require_device", lambda *t: None)
    for name, f in (("paged_attention", attention), ("paged_append", append), ("paged_append_packed", packed), ("paged_slots", slots),
                    ("paged_bounds", bounds), ("paged_select", ref.select), ("paged_sparse_attention", sparse)):
        monkeypatch.setattr(paged, name, f)
    return paged


@pytest.mark.parametrize("code", [E4, I8], ids=["e4m3", "int8"])
@pytest.mark.parametrize("select", [None, 2])
def test_cache_in_8_bits(plain, code, select):
    g = torch.Generator().manual_seed(1)
    c = plain.PagedIclKVCache(3, 2, 2, 32, 100, 16, 16, code, "cpu", select=select)
    held = [[] for _ in range(3)]
    for i, new in enumerate(([20, 1, 0], [1, 1, 1], [15, 40, 16], [0, 0, 0])):
        for b in range(2):
            rows = [torch.randn(r, 2, 2, 32, generator=g) for r in new]
            if i == 2:
                x = torch.cat(rows)
                c.append_packed(b, x[:, 0], x[:, 1], new)
            else:
                x = torch.nn.utils.rnn.pad_sequence(rows, batch_first=True).permute(2, 0, 3, 1, 4)
                c.append(b, x[0].to(BF) if i == 1 else x[0], x[1].to(BF) if i == 1 else x[1], new)
            if b == 1:
                for s in range(3):
                    held[s].append(rows[s])
    assert c.lengths.tolist() == [[36, 42, 17]] * 2
    assert (c.scales[:, c.table[c.table >= 0].long()] > 0).all()
    for dtype in (F32, BF):
        q = torch.randn(3, 2, 4, 32, generator=g).to(dtype)
        out = c.query(1, q)
        assert out.dtype == dtype
        if select is None:
            for s in range(3):
                kv = torch.cat(held[s])
                p = torch.softmax(torch.einsum("htd,rhd->htr", q[s].float(), kv[:, 0]) * 32 ** -0.5, -1)
                assert (out[s].float() - torch.einsum("htr,rhd->htd", p, kv[:, 1])).abs().max() < 0.3
        else:
            index = ref.select(q, c.bounds[1], c.bound_scales[1], c.table, c.lengths[1], 16, 2)
            o, _ = ref.sparse_attention(q, ref.values(c.keys[1], c.scales[1], 0), ref.values(c.values[1], c.scales[1], 1), c.table,
                                        c.lengths[1], index, 32 ** -0.5)
            assert torch.equal(out, o.to(dtype))
            assert torch.equal(c.estimators(1, 3).query(1, q[1:]), out[1:])


def test_cache_refuses(plain):
    for kw, word in ((dict(dtype=E4, track=True), "tracks no weights"), (dict(select=3, track=True), "tracks no weights"),
                     (dict(select=0), "at least 1")):
        with pytest.raises(ValueError, match=word):
            plain.PagedIclKVCache(2, 1, 2, 32, 64, 9, 16, kw.pop("dtype", F32), "cpu", **kw)
    c = plain.PagedIclKVCache(2, 1, 2, 32, 64, 9, 16, I8, "cpu")
    k = torch.zeros(2, 2, 3, 32)
    with pytest.raises(ValueError, match="cast before"):
        c.append(0, k.half(), k.half())
    with pytest.raises(ValueError, match="cast before"):
        c.append(0, k, k.to(BF))
    with pytest.raises(ValueError, match="evict needs"):
        c.evict(3)
    for rows, total in (([1, 2, 3], 6), ([1, -1], 0), ([2, 2], 3)):
        with pytest.raises(ValueError, match="rows must|append_packed expects"):
            c.append_packed(0, torch.zeros(total, 2, 32), torch.zeros(total, 2, 32), rows)
    assert c.free_pages == 9
    c.append(0, k, k)
    with pytest.raises(ValueError, match="wider"):
        c.query(0, torch.zeros(2, 2, 1, 32, dtype=torch.float64))
    with pytest.raises(ValueError, match="queries only"):
        c.estimators(0, 1).append_packed(0, k[:, :, 0], k[:, :, 0], [2])
    assert c.query(0, torch.zeros(2, 2, 1, 32, dtype=torch.float16)).dtype == F32
