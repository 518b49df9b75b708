"""`paged.attention` of fp32 queries of any size over fp16 pages: beyond fp16's range, below it, and rows and heads of
very different sizes in one call."""
import pytest
import torch

import paged_oracle as oracle
from test_gpu_pages import F16, F32, setup

pytestmark = pytest.mark.gpu

SHAPES = [
    ([1, 1], [40, 9], 100, 4, 2, 64),                    # one launch
    ([1, 2], [700, 40], 4000, 4, 2, 128),                # parts that are joined
    ([1] * 60, [1 + i for i in range(60)], 5000, 28, 4, 128),
    ([1] * 70, [30 + i for i in range(70)], 5000, 14, 2, 64),
    ([300, 280], [330, 300], 70, 28, 4, 128),            # requests of many rows, in one walk
    ([200, 260], [230, 270], 0, 14, 2, 64),
    ([90, 120], [1400, 1300], 2000, 14, 2, 64),
]


def check(s, x, scale):
    from seedplane_b200 import paged
    pages, batch = setup(s)
    hd = x.shape[2]
    lse = torch.empty(x.shape[:2], device="cuda")
    got = paged.attention(pages, 0, batch, x, scale=scale, lse=lse)
    pages.status()
    ref, absum, size, ref_lse = oracle.attention(s, x, scale)
    # a query is held to 2^-22 of itself and 2^-39 of its row's largest: that times the keys' |k|, at most twice in a weight
    keys = torch.nan_to_num(s["k"].float()).abs().amax().double()
    floor = 2.0 ** -39 * x.abs().amax(-1).double() * keys * hd * scale
    off = oracle.attention_bounds(F32, F16, hd, s["prefix"] + max(s["len"]), absum, size, ref) + 4 * floor[..., None] * absum
    assert ((got.double() - ref).abs() <= off).all()
    assert ((lse.double() - ref_lse).abs() <= size * hd * 2.0 ** -22 + ref_lse.abs() * 2.0 ** -22 + floor + 1e-4).all()
    return got, ref


@pytest.mark.parametrize("q,lens,prefix,nh,nkv,hd", SHAPES)
@pytest.mark.parametrize("size", [1e-30, 1e-12, 1e-5, 1e5, 1e8, 1e30])
def test_queries_of_any_size(q, lens, prefix, nh, nkv, hd, size):
    """The scale brings the scores back to those of unit queries."""
    s = oracle.make_batch(q=q, lens=lens, prefix=prefix, page=64, nkv=nkv, hd=hd, dtype=F16)
    x = size * torch.randn(s["rows"], nh, hd, device="cuda", generator=torch.Generator("cuda").manual_seed(4))
    got, ref = check(s, x, float(torch.tensor(hd ** -0.5 / size, dtype=F32)))
    assert float((got.double() - ref).norm() / ref.norm()) < 1e-5


@pytest.mark.parametrize("q,lens,prefix,nh,nkv,hd", SHAPES)
def test_rows_of_different_sizes(q, lens, prefix, nh, nkv, hd):
    """Rows and heads from nothing to 1e30, and dims of one row 2^20 apart that weigh alike."""
    s = oracle.make_batch(q=q, lens=lens, prefix=prefix, page=64, nkv=nkv, hd=hd, dtype=F16)
    g = torch.Generator("cuda").manual_seed(5)
    x = torch.randn(s["rows"], nh, hd, device="cuda", generator=g)
    x *= 10.0 ** torch.randint(-30, 31, x.shape[:2], device="cuda", generator=g)[..., None]
    x[:, 0] = 0
    x[:, 1] = torch.randn(s["rows"], hd, device="cuda", generator=g)
    x[:, 1, ::2] *= 2.0 ** 20
    s["k"][:, :, 0, :, ::2] *= 2.0 ** -20                # head 1's kv head
    check(s, x, hd ** -0.5)


@pytest.mark.parametrize("q,lens,prefix,nh,nkv,hd", SHAPES)
def test_rows_whose_scores_vanish_beside_others(q, lens, prefix, nh, nkv, hd):
    """A scale for queries of 1e30, and rows of nothing or of 1e-30: every key they see weighs alike."""
    s = oracle.make_batch(q=q, lens=lens, prefix=prefix, page=64, nkv=nkv, hd=hd, dtype=F16)
    g = torch.Generator("cuda").manual_seed(7)
    x = 1e30 * torch.randn(s["rows"], nh, hd, device="cuda", generator=g)
    x[:, 0] = 0
    x[:, 1] *= 1e-30
    x[:, 1] *= 1e-30
    x[:, 2] = torch.finfo(F32).smallest_normal / 4
    check(s, x, float(torch.tensor(hd ** -0.5 / 1e30, dtype=F32)))
    check(s, x * 0, float(torch.finfo(F32).smallest_normal / 8))
    check(s, x * 0, 3e38)                                # and nothing by the largest scale
