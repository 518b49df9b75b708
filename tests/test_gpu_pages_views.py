"""Pages that are views of wider ones: `paged.append` and `paged.attention` over the first 64 dims of 128-dim pages, and
one batch used with both."""
import pytest
import torch

import paged_oracle as oracle
from test_gpu_pages import BF16, F16, F32, check_attention, rope_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt,cache", [(F16, F16), (BF16, BF16), (F32, F16)])
@pytest.mark.parametrize("q,lens,prefix,nh,nkv", [
    ([1, 1, 1], [70, 9, 130], 5000, 4, 2),
    ([1] * 40, [1 + 3 * i for i in range(40)], 5000, 28, 4),
    ([300, 1, 280], [330, 40, 300], 130, 14, 2),
])
def test_one_batch_over_pages_of_both_widths(q, lens, prefix, nh, nkv, dt, cache):
    from seedplane_b200 import paged
    s = oracle.make_batch(q=q, lens=lens, prefix=prefix, page=64, nkv=nkv, hd=128, dtype=cache)
    narrow = dict(s, k=s["k"][..., :64], v=s["v"][..., :64])
    batch = paged.PageBatch(s["tables"], s["lens"], q_start=s["q_start"], tokens=s["rows"], max_q=max(q),
                            prefix_table=s["prefix_table"], prefix_len=prefix)
    g = torch.Generator("cuda").manual_seed(9)
    for which in (narrow, s, narrow):                    # the same strides, the same batch
        pages = paged.PagedKV.wrap(which["k"], which["v"])
        x = (1.5 * torch.randn(s["rows"], nh, which["k"].shape[4], device="cuda", generator=g)).to(dt)
        got = paged.attention(pages, 0, batch, x)
        pages.status()
        check_attention(which, x, got)


def test_append_leaves_the_other_dims():
    from seedplane_b200 import paged
    s = oracle.make_batch(q=[3, 1], lens=[9, 40], prefix=0, page=16, nkv=2, hd=128, dtype=F16, garbage=5.0)
    old = s["k"].clone(), s["v"].clone()
    pages = paged.PagedKV.wrap(s["k"][..., :64], s["v"][..., :64])
    batch = paged.PageBatch(s["tables"], s["lens"], q_start=s["q_start"], tokens=4, max_q=3)
    qkv = torch.randn(4, 8 * 64, device="cuda").half()
    rope = rope_of(50, 64)
    paged.append(pages, 0, batch, qkv, 4, rope)
    pages.status()
    narrow = dict(s, k=s["k"][..., :64], v=s["v"][..., :64])
    positions = [lens - n + i for n, lens in ((3, 9), (1, 40)) for i in range(n)]
    ref, size = oracle.append(narrow, qkv, None, rope, positions, 4, 64, False)
    t = 0
    for b, (n, length) in enumerate(((3, 9), (1, 40))):
        for i in range(n):
            key = length - n + i
            k = s["k"][0, s["own"][b][key // 16], :, key % 16, :64].double()
            assert ((k - ref[t, 4:6]).abs() <= 2.0 ** -11 * ref[t, 4:6].abs() + 4 * 2.0 ** -24 * size[t, 4:6] + 2.0 ** -25).all()
            t += 1
    assert torch.equal(s["k"][..., 64:], old[0][..., 64:]) and torch.equal(s["v"][..., 64:], old[1][..., 64:])
