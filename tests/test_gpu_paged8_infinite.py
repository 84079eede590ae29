"""GPU tests of infinite queries over 8-bit pools: scores of -inf take no part, in fp32 (three bf16 terms a value) as in bf16."""
import math

import pytest
import torch

import paged8_ref as ref
from test_gpu_paged8 import BF, E4, F32, I8, _case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("code", [E4, I8], ids=["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("lengths", [[100, 33, 0], [2000, 300, 7]])
def test_infinite_queries(dev, dtype, code, lengths):
    import tabicl_mi355_paged as paged
    q, kp, vp, scales, table, n, g = _case(dev, 31, lengths, H=2, T=3, D=64, dtype=dtype, code=code)
    d, R = 5, kp.shape[2]
    one = torch.full((), 3.0, device=dev).to(code).view(torch.uint8)
    kp.view(torch.uint8)[..., d] = one  # dim d of every key is 3 codes
    q[0, 0, 0, d] = -math.inf      # every score -inf: 0
    q[0, 1, 1, d] = math.inf       # every score inf: NaN, as of inf - inf
    q[0, 0, 2, 9] = math.nan
    # one key of the other sign: the only score that is not -inf
    kp.view(torch.uint8)[table[1, 0].long(), 1, 4, d] = torch.full((), 0.0, device=dev).to(code).view(torch.uint8)
    q[1, 1, 1, d] = -math.inf
    clean = q.clone()
    clean[0, 0, 0], clean[0, 1, 1], clean[0, 0, 2], clean[1, 1, 1] = 0, 0, 0, 0
    out = paged.paged_attention(q, kp, vp, table, n, scales=scales)
    want = paged.paged_attention(clean, kp, vp, table, n, scales=scales)
    torch.cuda.synchronize()
    assert (out[0, 0, 0] == 0).all()
    assert torch.isnan(out[0, 1, 1]).all() and torch.isnan(out[0, 0, 2]).all()
    assert torch.isnan(out[1, 1, 1]).all()  # -inf times 0
    for i in range(2):
        for h in range(2):
            for t in range(3):
                if (i, h, t) not in ((0, 0, 0), (0, 1, 1), (0, 0, 2), (1, 1, 1)):
                    assert torch.equal(out[i, h, t], want[i, h, t])
    # a key of the other sign: its score is inf
    kp.view(torch.uint8)[table[1, 0].long(), 1, 4, d] = torch.full((), -3.0, device=dev).to(code).view(torch.uint8)
    assert torch.isnan(paged.paged_attention(q, kp, vp, table, n, scales=scales)[1, 1, 1]).all()
    # the list's form: a page of scores of -inf beside no other
    index = torch.zeros(3, 2, 3, 2, dtype=torch.int32, device=dev)
    index[..., 1] = -1
    few = paged.paged_sparse_attention(q, kp, vp, table, n, index, scales=scales)
    assert (few[0, 0, 0] == 0).all() and torch.isnan(few[0, 1, 1]).all()
    v = ref.values(vp, scales, 1)[table[0, 0].long(), 0, :min(lengths[0], R)]
    assert torch.isfinite(v).all()
