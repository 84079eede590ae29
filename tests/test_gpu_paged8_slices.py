"""GPU test of a query over selected pages with more rows than paged_select takes in a call: as the same rows in two queries."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.int8], ids=["bf16", "int8"])
def test_more_rows_than_a_call_takes(dev, dtype):
    import tabicl_mi355_paged as paged
    g = torch.Generator(device=dev).manual_seed(2)
    S, H, D, T = 2, 8, 32, 140000  # 2,240,000 query rows over sequences and heads
    c = paged.PagedIclKVCache(S, 1, H, D, 80, 10, 16, dtype, dev, select=2)
    k, v = (torch.randn(S, H, 80, D, generator=g, device=dev).to(torch.bfloat16) for _ in range(2))
    c.append(0, k, v, [80, 50])
    q = torch.randn(S, H, T, D, generator=g, device=dev).to(torch.bfloat16)
    out = c.query(0, q)
    half = T // 2 + 7
    for part in (slice(0, half), slice(half, T)):
        assert torch.equal(out[:, :, part], c.query(0, q[:, :, part]))
