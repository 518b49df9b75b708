"""`paged.attention` of scores of any size: the keys that share a row's largest score share its weight, whatever the
score, in every kernel and across key ranges that are joined."""
import pytest
import torch

import paged_oracle as oracle
from test_gpu_pages import BF16, F16, F32, setup

pytestmark = pytest.mark.gpu

SHAPES = [
    ([1, 1], [40, 9], 100, 4, 2, 64),                    # one launch
    ([1, 2], [700, 40], 4000, 4, 2, 128),                # parts that are joined
    ([1] * 60, [1 + i for i in range(60)], 5000, 28, 4, 128),
    ([1] * 70, [30 + i for i in range(70)], 5000, 14, 2, 64),
    ([300, 280], [330, 300], 70, 28, 4, 128),            # requests of many rows, in one walk
    ([90, 120], [1400, 1300], 2000, 14, 2, 64),
]


@pytest.mark.parametrize("q,lens,prefix,nh,nkv,hd", SHAPES)
@pytest.mark.parametrize("dt,cache,large", [(F16, F16, 3.0e4), (BF16, BF16, 1.0e14), (F32, F16, 3.0e4), (F32, F16, 50.0),
                                            (F32, F16, 32768.0)])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_of_any_size(q, lens, prefix, nh, nkv, hd, dt, cache, large, sign):
    from seedplane_b200 import paged
    s = oracle.make_batch(q=q, lens=lens, prefix=prefix, page=64, nkv=nkv, hd=hd, dtype=cache, garbage=0.0)
    g = torch.Generator("cuda").manual_seed(12)
    # one dim counts, so that every score is exact in 32 bits: a few of eight sizes, or their negatives
    size = large * (1 + torch.randint(0, 8, s["k"].shape[:4], device="cuda", generator=g) / 8)
    s["k"].zero_()
    s["k"][..., 3] = (sign * size).to(cache)
    x = torch.zeros(s["rows"], nh, hd, device="cuda")
    x[..., 3] = large * (1 + torch.randint(0, 64, x.shape[:2], device="cuda", generator=g) / 64)
    x = x.to(dt)
    pages, batch = setup(s)
    for scale in (None, 0.37):
        lse = torch.empty(s["rows"], nh, device="cuda")
        got = paged.attention(pages, 0, batch, x, scale=scale, lse=lse)
        pages.status()
        ref, absum, _, ref_lse = oracle.attention(s, x, scale or hd ** -0.5)
        if dt == F32 and large == 3.0e4:
            # these queries have more than 11 bits, and q k, the sum of their two halves' products, more than 24: scores of
            # 1e9 are off by 2^-23 of themselves, 100, by the order of the sums, which differs from kernel to kernel; so
            # the largest need not share the weight evenly. The values lie between the least and the largest all the same
            off = torch.full_like(ref, float(s["v"].max() - s["v"].min()))
        elif large > 1e4:                                # equal weights: exact but for sums, the quotient and the output
            off = torch.finfo(dt).eps / 2 * ref.abs() + 2.0 ** -18 * absum
        else:                                            # scores of 2,500 to 3.4e5: off by 2^-24 of their differences twice
            score = 2 * 2.0 ** -24 * 2 * large * large * 4
            off = torch.finfo(dt).eps / 2 * ref.abs() + (2.0 ** -18 + 2 * score) * absum
        assert ((got.double() - ref).abs() <= off).all()
        assert ((lse.double() - ref_lse).abs() <= 4 * 2.0 ** -24 * ref_lse.abs() + 1e-5).all()
