"""`paged.attention` of queries that hold a NaN: NaN in that (row, head)'s values and log-sum-exp, nothing else touched."""
import math

import pytest
import torch

import paged_oracle as oracle
from test_gpu_pages import BF16, F16, F32, check_attention, run_attention, setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt,cache", [(F16, F16), (BF16, BF16), (F32, F16)])
@pytest.mark.parametrize("q,lens,prefix", [
    ([1, 1], [40, 9], 100),                              # one launch
    ([1, 1, 1], [700, 40, 5], 4000),                     # parts that are joined
    ([1] * 60, [1 + i for i in range(60)], 5000),        # the stacked rows of a batch
    ([300, 280], [330, 300], 70),                        # requests of many rows
])
def test_nan_queries(q, lens, prefix, dt, cache):
    from seedplane_b200 import paged
    s = oracle.make_batch(q=q, lens=lens, prefix=prefix, page=64, nkv=4, hd=128, dtype=cache)
    lse = torch.empty(s["rows"], 28, device="cuda")
    x, want = run_attention(s, 28, dt, lse=lse)
    check_attention(s, x, want, lse)
    bad = torch.zeros(x.shape[:2], dtype=torch.bool, device="cuda")
    for t, h in ((0, 0), (s["rows"] - 1, 27), (s["rows"] // 2, 13)):
        x[t, h, 5 + h] = math.nan
        bad[t, h] = True
    got_lse = torch.empty_like(lse)
    pages, batch = setup(s)
    got = paged.attention(pages, 0, batch, x, lse=got_lse)
    pages.status()
    assert torch.isnan(got[bad]).all() and torch.isnan(got_lse[bad]).all()
    assert torch.equal(got[~bad], want[~bad]) and torch.equal(got_lse[~bad], lse[~bad])
