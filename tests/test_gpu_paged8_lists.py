"""GPU tests of attention over lists of pages of an 8-bit pool, whose lists name pages that hold no rows of the sequence: given
out but not filled, so that nobody has written their scales."""
import math

import pytest
import torch

import paged8_ref as ref
import paged_ref
from test_gpu_paged8 import BF, E4, F32, I8
from test_gpu_sparse import _case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale", [math.nan, math.inf, -math.inf], ids=["nan", "inf", "-inf"])
@pytest.mark.parametrize("fmt", [E4, I8], ids=["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("D,R,T,K", [(64, 16, 1, 6), (64, 32, 2, 9), (32, 64, 1, 40), (128, 16, 3, 90), (128, 256, 1, 5)])
def test_listed_pages_without_rows(dev, dtype, fmt, scale, D, R, T, K):
    # pages at and past the length beside pages with rows: in one turn with them, alone in a turn, behind the first 64 of a list
    import tabicl_mi355_paged as paged
    lengths = [5 * R, 0, 3, 2 * R + 1]
    q, kp, vp, scales, table, n, g = _case(dev, D + R, lengths, H=2, G=2, D=D, R=R, T=T, fmt=fmt, dtype=dtype, slack=2)
    for i, length in enumerate(lengths):
        scales[table[i, -(-length // R):].long()] = scale
    M = table.shape[1]
    index = torch.randint(0, M, (4, 2, T, K), generator=g, device=dev, dtype=torch.int32)
    index[0, 0, 0, :4] = torch.tensor([0, M - 1, M - 2, 1], dtype=torch.int32)
    index[0, 1] = M - 1  # nothing but pages without rows
    print(f"[sparse] pages without rows {fmt} {dtype} D {D} R {R} K {K}", flush=True)
    out = paged.paged_sparse_attention(q, kp, vp, table, n, index, scales=scales)
    torch.cuda.synchronize()
    want, tol = ref.sparse_attention(q, ref.values(kp, scales, 0), ref.values(vp, scales, 1), table, n, index, D ** -0.5)
    paged_ref.near(out, want, tol, "pages without rows")
    assert (out[1] == 0).all() and (out[0, 2:] == 0).all()
