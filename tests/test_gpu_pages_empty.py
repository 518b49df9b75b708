"""Rows that see no key among rows that do, where a request brings many tokens: `paged.attention` gives them zeros and
a log-sum-exp of -inf, whatever the queries hold."""
import pytest
import torch

import paged_oracle as oracle
from test_gpu_pages import BF16, F16, F32, check_attention, run_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt,cache", [(F16, F16), (BF16, BF16), (F32, F16)])
@pytest.mark.parametrize("nh,nkv,hd", [(28, 4, 128), (14, 2, 64)])
@pytest.mark.parametrize("q,lens", [
    ([300, 260, 310], [300, 0, 350]),                    # a request without any key
    ([400, 330, 1], [400, 20, 0]),                       # and one whose first rows come before its keys
    ([290, 280], [0, 0]),                                # nobody has a key
    ([30, 280, 40], [60, 0, 40]),
])
def test_packed_prompts_of_requests_without_keys(q, lens, nh, nkv, hd, dt, cache):
    s = oracle.make_batch(q=q, lens=lens, prefix=0, page=64, nkv=nkv, hd=hd, dtype=cache, tail_rows=2)
    lse = torch.full((s["rows"], nh), 5.0, device="cuda")
    out = torch.full((s["rows"], nh, hd), 7.0, device="cuda", dtype=dt)
    for seed in range(4):
        x, got = run_attention(s, nh, dt, out=out, lse=lse, seed=seed)
        check_attention(s, x, got, lse)
        for b, n in enumerate(q):                        # exact zeros, not small numbers
            blind = slice(s["start"][b], s["start"][b] + max(0, n - lens[b]))
            assert (got[blind] == 0).all() and torch.isneginf(lse[blind]).all()
        assert (got[s["start"][-1]:] == 7.0).all() and (lse[s["start"][-1]:] == 5.0).all()
