"""GPU tests of how many rows paged_reserve grants, against rows counted one by one: the page that the first of them joins may be
missing, in both forms of the kernel (one launch, two)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
I32 = torch.int32


def _granted(table, lengths, count, pages, R):
    """The new rows of each request up to the first that has no page, from a table with its pages given out."""
    out = []
    for row, length, add in zip(table, lengths, count):
        length = max(0, min(length, len(row) * R))
        t = 0
        while t < add and (length + t) // R < len(row) and 0 <= row[(length + t) // R] < pages:
            t += 1
        out.append(t)
    return out


@pytest.mark.parametrize("N", [6, 300])
@pytest.mark.parametrize("R", [16, 64])
def test_own_page_missing(dev, N, R):
    # lengths inside a page that the table does not have (in every way it may not), on an edge, in a page that is there
    import tabicl_mi355_paged as paged
    M, P = 5, 4 * N + 7
    table = torch.full((N, M), -1, dtype=I32)
    lengths, count = [], []
    for n in range(N):
        table[n, 0] = n
        lengths.append([R // 2 + 1, R + 3, R, 2 * R - 1, R + 1, 3 * R + 5][n % 6])
        count.append([5, 7, R + 2, 1, 0, 4 * R][n % 6])
        table[n, 1] = [-1, P, N + n, -1, -(2 ** 31), 2 ** 31 - 1][n % 6]
    table, n = table.to(dev), torch.tensor(lengths, dtype=I32, device=dev)
    new = torch.tensor(count, dtype=I32, device=dev)
    free = torch.arange(P, dtype=I32, device=dev)
    free[:2 * N] = torch.arange(2 * N, 4 * N, device=dev)
    fc = torch.tensor([2 * N], dtype=I32, device=dev)
    print(f"[books] own page missing N {N} R {R}", flush=True)
    granted = paged.paged_reserve(table, n, new, free, fc, R)
    slots, starts = paged.paged_slots(table, n, new, sum(count), P, R)
    torch.cuda.synchronize()
    assert granted.tolist() == _granted(table.tolist(), lengths, count, P, R)
    s, at = slots.tolist(), starts.tolist()
    for i, t in enumerate(granted.tolist()):  # as the slots have it
        rows = s[at[i]:at[i + 1]]
        assert all(x >= 0 for x in rows[:t]) and (t == len(rows) or rows[t] < 0)


def test_two_pages_of_none(dev):
    import tabicl_mi355_paged as paged
    table = torch.full((1, 2), -1, dtype=I32, device=dev)
    n, new = torch.tensor([10], dtype=I32, device=dev), torch.tensor([5], dtype=I32, device=dev)
    free, fc = torch.zeros(4, dtype=I32, device=dev), torch.tensor([4], dtype=I32, device=dev)
    assert paged.paged_reserve(table, n, new, free, fc, 16).tolist() == [0]
    assert table.tolist() == [[-1, -1]] and int(fc) == 4
