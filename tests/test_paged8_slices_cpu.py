"""CPU tests of queries over selected pages in slices: every query row of every sequence is answered once, whatever the limits, with
the plain forms in the kernels' place."""
import pytest
import torch

from test_paged8_cpu import BF, E4, I8, plain  # noqa: F401


@pytest.mark.parametrize("code", [E4, I8], ids=["e4m3", "int8"])
@pytest.mark.parametrize("rows,sparse,nbytes", [(1 << 21, 1 << 22, 1 << 30), (14, 1 << 22, 1 << 30), (4, 1 << 22, 1 << 30), (2, 4, 1 << 30),
                                                (1 << 21, 8, 1 << 30), (1 << 21, 36, 1 << 30), (1 << 21, 1 << 22, 200),
                                                (1 << 21, 1 << 22, 1), (26, 1 << 22, 1 << 30)])
def test_slices_cover_every_row(plain, monkeypatch, code, rows, sparse, nbytes):  # noqa: F811
    g = torch.Generator().manual_seed(3)
    S, H, G, T, D = 3, 2, 2, 5, 32
    c = plain.PagedIclKVCache(S, 1, H, D, 100, 21, 16, code, "cpu", select=2)
    k, v = (torch.randn(S, H, 90, D, generator=g) for _ in range(2))
    c.append(0, k, v, [90, 10, 50])
    q = torch.randn(S, G * H, T, D, generator=g)
    want = c.query(0, q)
    monkeypatch.setattr(plain, "_SELECT_ROWS", rows)
    monkeypatch.setattr(plain, "_SPARSE_ROWS", sparse)
    monkeypatch.setattr(plain, "_SELECT_BYTES", nbytes)
    seen = torch.zeros(S, T)
    select, attend = plain.paged_select, plain.paged_sparse_attention

    def counted(part, bnd, bs, table, *a):
        n, hq, t, _ = part.shape
        assert n * H * t <= rows and n * hq * t <= sparse and table.shape[0] == n
        assert 4 * n * H * t * 2 <= nbytes or n * t == 1
        return select(part, bnd, bs, table, *a)

    def marked(part, *a, **kw):
        for s in range(S):
            for t in range(T):
                if any(torch.equal(part[i, :, j], q[s, :, t]) for i in range(part.shape[0]) for j in range(part.shape[2])):
                    seen[s, t] += 1
        return attend(part, *a, **kw)

    monkeypatch.setattr(plain, "paged_select", counted)
    monkeypatch.setattr(plain, "paged_sparse_attention", marked)
    assert torch.equal(c.query(0, q), want)
    assert (seen == 1).all()
    out = torch.zeros(S, T, G * H, D).transpose(1, 2)
    assert c.query(0, q, out=out) is out and torch.equal(out, want)
    over = q.clone()
    assert torch.equal(c.query(0, over, out=over), want)
    # out in the queries' storage, not in their order
    both = torch.zeros(S * G * H * T * D)
    x = both.view(S, G * H, T, D).copy_(q)
    assert torch.equal(c.query(0, x, out=both.view(T, S, G * H, D).permute(1, 2, 0, 3)), want)
    assert c.query(0, q[:, :, :0]).shape == (S, G * H, 0, D)


def test_workspace_counts(plain, monkeypatch):  # noqa: F811
    # a table of more pages than fit in LDS: selection's workspace is part of what a slice holds
    import tabicl_mi355_native as nat
    S, H, D = 2, 2, 32
    c = plain.PagedIclKVCache(S, 1, H, D, 33000 * 16, 40, 16, I8, "cpu", select=3)
    x = torch.randn(S, H, 64, D).to(BF)
    c.append(0, x, x)
    each = nat.load().tabicl_paged_select_workspace_bytes(1, H, 1, 33000)
    assert each == 4 * H * 33000
    monkeypatch.setattr(c, "_capturing", lambda: True)  # the whole table, as a captured query has it
    monkeypatch.setattr(plain, "_SELECT_BYTES", 4 * (each + 4 * H * 3))
    calls = []

    def select(part, bnd, bs, table, lengths, R, K):
        calls.append(tuple(part.shape))
        return torch.zeros(part.shape[0], H, part.shape[2], K, dtype=torch.int32)

    monkeypatch.setattr(plain, "paged_select", select)
    monkeypatch.setattr(plain, "paged_sparse_attention", lambda q, *a, **kw: a[6] if a[6] is not None else torch.empty_like(q))
    c.query(0, torch.randn(S, H, 9, D).to(BF))
    assert sum(a * b for a, _, b, _ in calls) == S * 9 and all(a * b <= 4 for a, _, b, _ in calls)
