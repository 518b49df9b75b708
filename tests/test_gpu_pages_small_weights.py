"""`paged.attention` where one key takes nearly all of a row's weight and its value is 0, so that thousands of small
weights make the output: fp16 probabilities keep their bits below the largest one's."""
import pytest
import torch

import paged_oracle as oracle
from test_gpu_pages import BF16, F16, F32, setup

pytestmark = pytest.mark.gpu

# q lens, own lens, prefix, nh, nkv, hd: few rows, the stacked rows of a batch, a request of many rows after no prefix
# and after a prefix (parts or one walk)
SHAPES = [
    ([1, 1], [70, 9], 4096, 4, 2, 128),
    ([1, 2], [700, 40], 4000, 4, 2, 64),
    ([1] * 12, [5 + 3 * i for i in range(12)], 6000, 28, 4, 128),
    ([1] * 60, [1 + i % 40 for i in range(60)], 5000, 14, 2, 64),
    ([1] * 50, [1 + 2 * i for i in range(50)], 5000, 28, 4, 128),
    ([150], [2600], 0, 14, 2, 64),
    ([30, 70], [2100, 70], 3000, 28, 4, 128),
    ([160, 190, 140, 220], [300, 190, 900, 240], 2500, 28, 4, 128),
]


@pytest.mark.parametrize("q,lens,prefix,nh,nkv,hd", SHAPES)
@pytest.mark.parametrize("dt,cache", [(F16, F16), (BF16, BF16), (F32, F16)])
@pytest.mark.parametrize("height", [11.5, 15.5, 17.0, 19.5])
@pytest.mark.parametrize("flat", [False, True])
def test_small_weights_behind_a_large_one(q, lens, prefix, nh, nkv, hd, dt, cache, height, flat):
    from seedplane_b200 import paged
    s = oracle.make_batch(q=q, lens=lens, prefix=prefix, page=64, nkv=nkv, hd=hd, dtype=cache, garbage=0.0)
    if flat:                                             # equal small weights: their roundings add up
        s["k"].zero_()
        s["v"].abs_()
    s["k"][..., 0] = 0
    owner = s["prefix_pages"] or s["own"][0]
    sinks = [(owner[0], 0), (owner[(prefix or lens[0]) // 64 - 1], 63)]
    for page, slot in sinks[:1] if height > 16 else sinks[1:]:       # before the others, or behind most
        s["k"][0, page, :, slot] = 0
        s["k"][0, page, :, slot, 0] = 8
        s["v"][0, page, :, slot] = 0
    pages, batch = setup(s)
    g = torch.Generator("cuda").manual_seed(6)
    x = torch.randn(s["rows"], nh, hd, device="cuda", generator=g)
    x[..., 0] = height * hd ** 0.5 / 8
    x = x.to(dt)
    got = paged.attention(pages, 0, batch, x)
    pages.status()
    ref, absum, size, _ = oracle.attention(s, x, hd ** -0.5)
    off = oracle.attention_bounds(dt, cache, hd, prefix + max(lens), absum, size, ref)
    # fp16's subnormals round by 2^-25, and a row's largest probability is held at 2^11 (fp32 queries) or 2^7 at least:
    # that share of sum |v| over the keys a row sees (its largest probability is below 1)
    if cache == F16:
        values = torch.zeros_like(ref)
        for b, n in enumerate(q):
            v = oracle.keys_of(s, b, "v").abs().cumsum(1)
            for i in range(n):
                m = prefix + lens[b] - n + i + 1
                values[s["start"][b] + i] = v[:, m - 1].repeat_interleave(nh // nkv, 0)
        off = off + 2.0 ** (-36 if dt == F32 else -32) * values
    assert ((got.double() - ref).abs() <= off).all()
    if dt == F32:
        # in all: the roundings of different small weights are independent of one another (2^-36 a key against 2^-28, the
        # least weight here, over the root of thousands of keys), those of equal ones the same
        assert float((got.double() - ref).norm() / ref.norm()) < (2.0 ** -7 if flat else 2.0 ** -9)
