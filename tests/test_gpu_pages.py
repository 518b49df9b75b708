"""Paged K / V on the GPU (`paged.append`, `paged.attention`): against the formulas in 64 bits at ragged
lengths, page sizes that end inside a tile, every type and layout, garbage (NaN) in every slot that no
key owns, bad tables, captured graphs, and the two together with `speculative.accept_chains`."""
import math

import pytest
import torch

import paged_oracle as oracle

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def setup(s, max_q=None, ragged=True):
    from seedplane_b200 import paged
    pages = paged.PagedKV.wrap(s["k"], s["v"])
    batch = paged.PageBatch(s["tables"], s["lens"], q_start=s["q_start"] if ragged else None, tokens=s["rows"],
                            max_q=max_q or max(s["q"] + [1]), prefix_table=s["prefix_table"], prefix_len=s["prefix"])
    return pages, batch


def bits(t):
    return t.contiguous().view(torch.int16 if t.element_size() == 2 else torch.int32)


def rope_of(positions, rot, seed=3):
    a = torch.arange(positions, dtype=torch.float64)[:, None] * (1e4 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot))
    return torch.stack((a.cos(), a.sin()), -1).float().cuda()


# ---- append ------------------------------------------------------------------------------------
APPEND = [
    # q lens, own lens, prefix, page, nh, nkv, hd, rows, cache, rot, interleaved, bias
    ([1], [1], 0, 16, 14, 2, 64, F32, F16, 64, False, True),
    ([1, 1, 1], [5, 64, 65], 100, 64, 28, 4, 128, F32, F16, 128, False, True),
    ([3, 0, 7, 1], [3, 9, 40, 33], 17, 16, 12, 2, 128, F16, F16, 128, False, False),
    ([2, 5], [20, 21], 5, 5, 4, 4, 64, BF16, BF16, 32, True, True),
    ([4, 9], [4, 30], 0, 32, 6, 3, 128, BF16, BF16, 64, True, False),
    ([33], [70], 3, 128, 3, 1, 64, F32, BF16, 64, True, True),
    ([6, 2], [19, 2], 31, 7, 5, 1, 128, F32, F16, 20, False, True),    # rot_dim no multiple of 16
    ([6, 2], [19, 2], 31, 1, 5, 1, 64, F16, F16, 2, True, False),
]


@pytest.mark.parametrize("q,lens,prefix,page,nh,nkv,hd,dt,cache,rot,inter,bias", APPEND)
@pytest.mark.parametrize("odd", [False, True])
def test_append_matches_64_bits(q, lens, prefix, page, nh, nkv, hd, dt, cache, rot, inter, bias, odd):
    from seedplane_b200 import paged
    s = oracle.make_batch(q=q, lens=lens, prefix=prefix, page=page, nkv=nkv, hd=hd, dtype=cache, tail_rows=2, nhd=odd)
    pages, batch = setup(s)
    g = torch.Generator("cuda").manual_seed(1)
    cols = (nh + 2 * nkv) * hd
    wide = torch.randn(s["rows"], cols + (3 if odd else 0), device="cuda", generator=g).to(dt)
    qkv = wide[:, odd * 3:]                                          # odd: rows that are not 16-byte aligned
    b = torch.randn(cols, device="cuda", generator=g) if bias else None
    rope = rope_of(prefix + max(lens) + 40, rot)
    own = [prefix + lens[r] - n + i for r, n in enumerate(q) for i in range(n)]
    positions = [p + 31 for p in own] if odd else own
    given = torch.tensor(positions + [0, 0], dtype=torch.int32, device="cuda") if odd else None
    q_out = torch.full((s["rows"], nh, hd), 7.0, device="cuda", dtype=dt)
    before = [bits(s["k"]).clone(), bits(s["v"]).clone()]
    got = paged.append(pages, 0, batch, qkv, nh, rope, bias=b, interleaved=inter, positions=given, q_out=q_out)
    pages.status()
    assert got is q_out
    ref, size = oracle.append(s, qkv, b, rope, positions, nh, rot, inter)
    # one rounding to the output's type, and up to four of 2^-24 before it (bias, two products, a sum)
    off = lambda t: torch.finfo(t).eps / 2 * ref.abs() + 4 * 2.0 ** -24 * size + (2.0 ** -25 if t == F16 else 0)  # noqa: E731
    n = s["start"][-1]
    assert ((got[:n].double() - ref[:, :nh]).abs() <= off(dt)[:, :nh]).all()
    assert (got[n:] == 7.0).all()                                    # rows behind the last request
    touched = torch.zeros(s["k"].shape[1], nkv, page, dtype=torch.bool, device="cuda")
    for r, m in enumerate(q):
        for i in range(m):
            key, t = lens[r] - m + i, s["start"][r] + i
            p, j = s["own"][r][key // page], key % page
            touched[p, :, j] = True
            for which, h0 in (("k", nh), ("v", nh + nkv)):
                assert ((s[which][0, p, :, j].double() - ref[t, h0:h0 + nkv]).abs() <= off(cache)[t, h0:h0 + nkv]).all()
    for which, old in zip(("k", "v"), before):
        same = (bits(s[which]) == old.view(s[which].shape)).all(-1)[0]
        assert same[~touched].all()


def test_append_records_bad_pages_lengths_and_positions():
    from seedplane_b200 import paged
    from seedplane_b200._native import EngineError
    s = oracle.make_batch(q=[1, 1, 1, 1], lens=[4, 4, 4, 4], prefix=0, page=16, nkv=1, hd=64, dtype=F16, garbage=0.0)
    pages, batch = setup(s)
    rope, qkv = rope_of(8, 64), torch.ones(4, 4 * 64, device="cuda")
    paged.append(pages, 0, batch, qkv, 2, rope)
    pages.status()
    for change in ("page", "page", "length", "length", "position"):
        tables, lens = s["tables"].clone(), s["lens"].clone()
        positions = None
        if change == "page":
            s["tables"][2, 0] = s["k"].shape[1] if tables[2, 0] >= 0 else -1
        elif change == "length":
            s["lens"][1] = 0 if lens[3] == 4 else 17
        else:
            positions = torch.tensor([0, 8, -1, 3], dtype=torch.int32, device="cuda")
        s["k"].zero_()
        paged.append(pages, 0, batch, qkv, 2, rope, positions=positions)
        with pytest.raises(EngineError):
            pages.status()
        pages.status()                                               # cleared
        written = int((s["k"] != 0).any(-1).sum())
        assert written == (4 if change == "position" else 3)
        s["tables"].copy_(tables)
        s["lens"].copy_(lens)


# ---- attention ---------------------------------------------------------------------------------
ATTENTION = [
    # q lens, own lens, prefix, page, nh, nkv, hd
    ([1], [1], 0, 16, 14, 2, 64),
    ([1], [1], 1, 16, 4, 4, 64),
    ([1, 1, 1], [1, 300, 17], 513, 64, 12, 2, 128),
    ([1, 0, 1, 1, 1], [90, 40, 1, 129, 1000], 200, 16, 28, 4, 128),
    ([5, 1, 3], [5, 64, 128], 300, 32, 14, 2, 64),
    ([4, 2], [260, 2], 0, 128, 28, 4, 128),
    ([70, 33, 1], [70, 200, 9], 190, 64, 12, 2, 128),
    ([40, 130], [300, 131], 1000, 256, 14, 2, 64),
    ([3, 2], [30, 31], 45, 5, 6, 3, 128),                            # a page size that divides no tile
    ([1] * 40, list(range(1, 41)), 700, 64, 7, 1, 128),
    ([1] * 37, [2] * 37, 2500, 128, 14, 2, 64),
    ([2, 1], [3, 1], 5, 1, 4, 1, 64),
    ([1, 1], [0, 0], 33, 16, 4, 2, 64),                              # rows that see the prefix alone
    ([2, 1], [1, 0], 0, 16, 4, 2, 128),                              # rows that see nothing
]


def run_attention(s, nh, dt, scale=None, ragged=True, spread=1.5, out=None, lse=None, seed=4):
    from seedplane_b200 import paged
    pages, batch = setup(s, ragged=ragged)
    g = torch.Generator("cuda").manual_seed(seed)
    hd = s["k"].shape[4]
    q = (spread * torch.randn(s["rows"], nh, hd, device="cuda", generator=g)).to(dt)
    got = paged.attention(pages, 0, batch, q, scale=scale, out=out, lse=lse)
    pages.status()
    return q, got


def check_attention(s, q, got, lse=None, scale=None):
    hd = q.shape[2]
    scale = hd ** -0.5 if scale is None else scale
    ref, absum, size, ref_lse = oracle.attention(s, q, scale)
    keys = s["prefix"] + max(s["len"])
    n = s["start"][-1]
    off = oracle.attention_bounds(q.dtype, s["k"].dtype, hd, keys, absum, size, ref)
    assert ((got[:n].double() - ref).abs() <= off).all()
    if q.dtype == F32 and float(ref.norm()):
        assert float((got[:n].double() - ref).norm() / ref.norm()) < 1e-5
    if lse is not None:
        seen = torch.isfinite(ref_lse)
        assert torch.equal(torch.isneginf(lse[:n]), ~seen)
        assert ((lse[:n].double() - ref_lse).abs()[seen] <= (size * hd * 2.0 ** -22 + ref_lse.abs() * 2.0 ** -22 + 1e-4)[seen]).all()


@pytest.mark.parametrize("q,lens,prefix,page,nh,nkv,hd", ATTENTION)
@pytest.mark.parametrize("dt,cache", [(F16, F16), (BF16, BF16), (F32, F16)])
def test_attention_matches_64_bits(q, lens, prefix, page, nh, nkv, hd, dt, cache):
    s = oracle.make_batch(q=q, lens=lens, prefix=prefix, page=page, nkv=nkv, hd=hd, dtype=cache, tail_rows=3)
    lse = torch.full((s["rows"], nh), 5.0, device="cuda")
    out = torch.full((s["rows"], nh, hd), 7.0, device="cuda", dtype=dt)
    x, got = run_attention(s, nh, dt, out=out, lse=lse)
    assert got is out
    check_attention(s, x, got, lse)
    n = s["start"][-1]
    assert (got[n:] == 7.0).all() and (lse[n:] == 5.0).all()


@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("prefix,batch", [(4000, 3), (9000, 30), (300, 90)])
def test_attention_of_larger_batches_strides_and_scales(dt, prefix, batch):
    s = oracle.make_batch(q=[1] * batch, lens=[1 + (37 * i) % 400 for i in range(batch)], prefix=prefix, page=64, nkv=2, hd=128,
                          dtype=F16, nhd=True)                       # slots before heads: other strides
    g = torch.Generator("cuda").manual_seed(2)
    from seedplane_b200 import paged
    pages, b = setup(s, ragged=False)
    wide = torch.randn(batch, 18, 128, device="cuda", generator=g).to(dt)
    q = wide[:, 2:14]
    got = paged.attention(pages, 0, b, q, scale=0.21)
    pages.status()
    check_attention(s, q, got, scale=0.21)


@pytest.mark.parametrize("dt,cache", [(F16, F16), (BF16, BF16), (F32, F16)])
@pytest.mark.parametrize("prefix", [1, 15, 16, 17, 127, 128, 129, 257])
def test_attention_of_short_prefixes_under_many_rows(prefix, dt, cache):
    for batch, nh, nkv, hd, page in ((40, 14, 2, 64, 16), (9, 12, 2, 128, 32), (23, 28, 4, 128, 8)):
        s = oracle.make_batch(q=[1] * batch, lens=[1 + (7 * i) % 33 for i in range(batch)], prefix=prefix, page=page, nkv=nkv, hd=hd,
                              dtype=cache, seed=prefix)
        x, got = run_attention(s, nh, dt)
        check_attention(s, x, got)


@pytest.mark.parametrize("dt,cache", [(F16, F16), (BF16, BF16), (F32, F16)])
@pytest.mark.parametrize("prefix", [64, 127, 129, 300])
def test_attention_of_hundreds_of_requests(prefix, dt, cache):
    """Enough rows for the tensor-core walk of a short prefix, and for the join of a row by one warp."""
    for batch, nh, nkv, hd, page in ((420, 14, 2, 64, 16), (200, 28, 4, 128, 32)):
        s = oracle.make_batch(q=[1] * batch, lens=[(5 * i) % 41 for i in range(1, batch + 1)], prefix=prefix, page=page, nkv=nkv,
                              hd=hd, dtype=cache, seed=prefix)
        lse = torch.empty(s["rows"], nh, device="cuda")
        x, got = run_attention(s, nh, dt, lse=lse)
        check_attention(s, x, got, lse)


@pytest.mark.parametrize("dt,cache", [(F16, F16), (BF16, BF16), (F32, F16)])
@pytest.mark.parametrize("prefix", [1800, 1919, 2049, 6001])
def test_attention_of_a_long_prefix_under_one_row_tile(prefix, dt, cache):
    for page in (8, 256):
        s = oracle.make_batch(q=[1] * 14, lens=[1 + 9 * i for i in range(14)], prefix=prefix, page=page, nkv=4, hd=128, dtype=cache,
                              seed=prefix)
        x, got = run_attention(s, 28, dt)
        check_attention(s, x, got)


@pytest.mark.parametrize("dt,cache,nh,nkv,hd", [(F16, F16, 28, 4, 128), (BF16, BF16, 14, 2, 64), (F32, F16, 12, 2, 128),
                                                (F32, F16, 16, 8, 64)])
@pytest.mark.parametrize("prefix,page", [(130, 64), (0, 16), (31, 128)])
def test_attention_of_packed_prompts(dt, cache, nh, nkv, hd, prefix, page):
    """Rows enough for a row tile to walk the prefix and its request's own keys by itself."""
    q = [300, 1, 250, 0, 420, 129, 512, 40]
    s = oracle.make_batch(q=q, lens=[n + (17 * i) % 90 for i, n in enumerate(q)], prefix=prefix, page=page, nkv=nkv, hd=hd, dtype=cache,
                          tail_rows=2)
    out = torch.full((s["rows"], nh, hd), 7.0, device="cuda", dtype=dt)
    lse = torch.full((s["rows"], nh), 5.0, device="cuda")
    x, got = run_attention(s, nh, dt, out=out, lse=lse)
    check_attention(s, x, got, lse)
    assert (got[s["start"][-1]:] == 7.0).all()


def test_attention_of_values_that_a_wrong_order_would_show():
    """Keys far apart in size and values that name their key: the row of the largest key comes back exactly."""
    for prefix, own in ((300, 40), (128, 200), (0, 77)):
        s = oracle.make_batch(q=[1, 1], lens=[own, own + 3], prefix=prefix, page=16, nkv=1, hd=64, dtype=F16, garbage=0.0)
        s["k"].zero_()
        s["v"].zero_()
        n = prefix + own
        for b in range(2):
            for j in range(prefix if b else 0, prefix + s["len"][b]):
                page = s["prefix_pages"][j // 16] if j < prefix else s["own"][b][(j - prefix) // 16]
                at = j % 16 if j < prefix else (j - prefix) % 16
                s["k"][0, page, 0, at, 0] = 100.0 if j == (37 * (b + 1)) % n else 0.0
                s["v"][0, page, 0, at] = float(j % 251)
        from seedplane_b200 import paged
        pages, batch = setup(s)
        x = torch.zeros(2, 2, 64, device="cuda", dtype=F16)
        x[:, :, 0] = 50.0
        got = paged.attention(pages, 0, batch, x)
        hot = [j for j in (37 % n, 74 % n)]
        if prefix == 0:
            assert (got[0] == float(hot[0] % 251)).all() and (got[1] == float(hot[1] % 251)).all()
        else:                                            # the second request's hot key may lie in the shared prefix
            check_attention(s, x, got)


def test_attention_of_large_scores_and_infinite_keys_out_of_sight():
    """Scores of several hundred (one key wins), and infinities in slots behind a request's last key."""
    s = oracle.make_batch(q=[1, 2, 1], lens=[40, 41, 42], prefix=130, page=16, nkv=2, hd=64, dtype=F16, garbage=float("inf"))
    x, got = run_attention(s, 4, F16, spread=60.0)
    assert torch.isfinite(got).all()
    ref = oracle.attention(s, x, 64 ** -0.5)[0]
    # scores of up to 2,000: exact to hd 2^-23 of sum |q k| (about 5,000 here): 0.04 in the exponent
    assert ((got.double() - ref).abs() <= 0.1 * ref.abs().amax()).all()
    assert float((got.double() - ref).norm() / ref.norm()) < 0.02


def test_attention_without_any_key_gives_zeros():
    from seedplane_b200 import paged
    pages = paged.PagedKV(1, 2, 64, 3, 16, device="cuda")
    batch = paged.PageBatch(torch.zeros(2, 0, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"))
    out, lse = torch.full((2, 4, 64), 7.0, device="cuda").half(), torch.full((2, 4), 7.0, device="cuda")
    got = paged.attention(pages, 0, batch, torch.ones(2, 4, 64, device="cuda").half(), out=out, lse=lse)
    pages.status()
    assert (got == 0).all() and torch.isneginf(lse).all()
    none = paged.PageBatch(torch.zeros(0, 1, dtype=torch.int32, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda"))
    assert paged.attention(pages, 0, none, torch.ones(0, 4, 64, device="cuda").half()).shape == (0, 4, 64)


def test_attention_records_bad_tables_and_goes_on():
    from seedplane_b200 import paged
    from seedplane_b200._native import EngineError
    s = oracle.make_batch(q=[1, 1, 1], lens=[50, 60, 20], prefix=100, page=16, nkv=1, hd=64, dtype=F16)
    pages, batch = setup(s)
    q = torch.randn(3, 4, 64, device="cuda").half()
    good = paged.attention(pages, 0, batch, q)
    pages.status()
    s["tables"][1, 2] = 10 ** 6
    got = paged.attention(pages, 0, batch, q)
    with pytest.raises(EngineError):
        pages.status()
    assert torch.equal(got[0], good[0]) and torch.equal(got[2], good[2])
    assert torch.isfinite(got).all()
    s["tables"][1, 2] = -1
    paged.attention(pages, 0, batch, q)
    with pytest.raises(EngineError):
        pages.status()
    s["lens"][2] = 10 ** 6
    paged.attention(pages, 0, batch, q)
    with pytest.raises(EngineError):
        pages.status()
    s["lens"][2] = -5
    paged.attention(pages, 0, batch, q)
    with pytest.raises(EngineError):
        pages.status()


def test_attention_is_deterministic_and_captures_into_graphs():
    """Two graphs over one set of arrays, replayed in turn and after the lengths grew; a side stream."""
    from seedplane_b200 import paged
    lens = [70, 200, 3, 129]
    s = oracle.make_batch(q=[1] * 4, lens=lens, prefix=600, page=32, nkv=2, hd=128, dtype=F16)
    pages, batch = setup(s)
    q = torch.randn(4, 12, 128, device="cuda").half()
    eager = paged.attention(pages, 0, batch, q)
    assert torch.equal(eager, paged.attention(pages, 0, batch, q))
    graphs, outs = [], []
    side = torch.cuda.Stream()
    for _ in range(2):
        out = torch.zeros_like(q)
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            paged.attention(pages, 0, batch, q, out=out)
        graphs.append(g)
        outs.append(out)
    for new in (lens, [60, 190, 1, 100]):
        s["lens"].copy_(torch.tensor(new, dtype=torch.int32))
        s["len"] = new
        want = paged.attention(pages, 0, batch, q)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = paged.attention(pages, 0, batch, q)
        side.synchronize()
        assert torch.equal(again, want)
        check_attention(s, q, want)


def test_append_attention_and_verification_together():
    """A round of drafted tokens for a batch after a shared prefix: append the drafts, attend, verify, keep what was accepted
    (lens), append the next round over the refused ones."""
    from seedplane_b200 import paged, speculative
    nh, nkv, hd, page, prefix, n, V = 6, 2, 64, 16, 77, 3, 501
    lens = [9, 30, 1]
    s = oracle.make_batch(q=[n + 1] * 3, lens=[m + 2 * (n + 1) for m in lens], prefix=prefix, page=page, nkv=nkv, hd=hd, dtype=F16)
    kept = list(lens)
    rope = rope_of(prefix + 80, hd)
    g = torch.Generator("cuda").manual_seed(8)
    for _ in range(2):
        s["len"] = [m + n + 1 for m in kept]
        s["lens"].copy_(torch.tensor(s["len"], dtype=torch.int32))
        pages, batch = setup(s)
        qkv = torch.randn(s["rows"], (nh + 2 * nkv) * hd, device="cuda", generator=g)
        x = paged.append(pages, 0, batch, qkv, nh, rope)
        got = paged.attention(pages, 0, batch, x)
        pages.status()
        check_attention(s, x, got)
        w = torch.randn(nh * hd, V, device="cuda", generator=g)
        target = (got.reshape(3, n + 1, -1) @ w).contiguous()
        drafts = target[:, :n].argmax(-1).int()
        draft = target[:, :n] + 0.5 * torch.randn(3, n, V, device="cuda", generator=g)
        u = torch.rand(3, n + 1, device="cuda", generator=g, dtype=torch.float64)
        tokens, accepted = speculative.accept_chains(target, draft, drafts, u, temperature=0.8)
        want = oracle.chains(target.cpu(), draft.cpu(), drafts.cpu(), u.cpu(), None, torch.full((3,), 0.8))
        assert tokens.tolist() == want[0] and accepted.tolist() == want[1]
        kept = [m + a + 1 for m, a in zip(kept, accepted.tolist())]
