"""Verification of a batch's draft chains on the GPU (`speculative.accept_chains`): the same tokens as the
rule on lists in 64 bits, over types, ragged counts, temperatures, filtered rows and odd vocabularies."""
import math

import pytest
import torch

import paged_oracle as oracle

pytestmark = pytest.mark.gpu


def case(B, n, V, dt, seed, spread=3.0, near=0.5):
    g = torch.Generator().manual_seed(seed)
    target = (spread * torch.randn(B, n + 1, V, generator=g)).to(dt)
    draft = (target[:, :n].float() + near * torch.randn(B, n, V, generator=g)).to(dt)
    gumbel = -torch.log(-torch.log(torch.rand(B, n, V, generator=g, dtype=torch.float64)))
    drafts = (draft.double() + gumbel).argmax(-1).int() if n else torch.zeros(B, 0, dtype=torch.int32)
    u = torch.rand(B, n + 1, generator=g, dtype=torch.float64)
    return target, draft, drafts, u


def run(target, draft, drafts, u, counts=None, temperature=None):
    from seedplane_b200 import speculative
    dev = lambda t: t if t is None or not isinstance(t, torch.Tensor) else t.cuda()  # noqa: E731
    tokens, accepted = speculative.accept_chains(dev(target), dev(draft), dev(drafts), dev(u), counts=dev(counts),
                                                 temperature=dev(temperature))
    return tokens.tolist(), accepted.tolist()


@pytest.mark.parametrize("B,n,V", [(1, 1, 1), (1, 4, 2), (3, 2, 7), (5, 3, 1000), (2, 5, 8192), (4, 2, 8193), (2, 3, 50001),
                                   (1, 4, 151936), (3, 0, 3333), (2, 64, 300)])
@pytest.mark.parametrize("dt", [torch.float32, torch.float16, torch.bfloat16])
def test_chains_match_the_rule(B, n, V, dt):
    g = torch.Generator().manual_seed(V + n)
    target, draft, drafts, u = case(B, n, V, dt, seed=V + B)
    temperature = 0.5 + torch.rand(B, generator=g)
    counts = torch.randint(0, n + 1, (B,), generator=g, dtype=torch.int32)
    for d in (draft, None):
        for c in (None, counts):
            for t in (None, temperature):
                assert run(target, d, drafts, u, c, t) == oracle.chains(target, d, drafts, u, c, t)


def test_many_requests_and_flat_rows():
    """Flat rows: every token's share is near the others', so a sum in fewer bits would move the draw."""
    for seed in range(3):
        target, draft, drafts, u = case(24, 3, 40000, torch.float32, seed=seed, spread=0.05, near=0.05)
        assert run(target, draft, drafts, u) == oracle.chains(target, draft, drafts, u, None, None)


def test_greedy_rows_take_the_first_maximum():
    target, draft, drafts, u = case(4, 3, 100, torch.float32, seed=5)
    target[0, 0, 30] = target[0, 0, 70] = 50.0
    drafts[0, 0] = 30
    target[1, 0, 20] = target[1, 0, 60] = 50.0
    drafts[1, 0] = 60                                    # not the first: refused
    drafts[2] = target[2, :3].argmax(-1).int()
    t = torch.tensor([0.0, 0.0, 0.0, 1.0])
    got = run(target, draft, drafts, u, None, t)
    assert got == oracle.chains(target, draft, drafts, u, None, t)
    assert got[1][0] >= 1 and got[1][1] == 0 and got[0][1][0] == 20 and got[1][2] == 3
    assert run(target, None, drafts, u, None, 0.0)[1][2] == 3


def test_filtered_infinite_and_empty_rows():
    target, draft, drafts, u = case(6, 2, 600, torch.float32, seed=9)
    target[0, :, 10:] = -math.inf                        # filtered to ten tokens
    drafts[0, 0] = 500                                   # a token of no weight
    target[1, 0] = -math.inf                             # nothing to accept or draw
    target[2, 0, 17] = math.inf                          # all the weight
    drafts[2, 0] = 17
    target[3, 0, :300] = math.nan                        # NaN weighs nothing
    drafts[3, 0] = 4
    draft[4, 0] = -math.inf                              # the drafter has no distribution: its token costs nothing
    drafts[5, 0] = 600                                   # outside the vocabulary
    got = run(target, draft, drafts, u)
    assert got == oracle.chains(target, draft, drafts, u, None, None)
    assert got[1][1] == 0 and got[0][1] == [-1, -1, -1]
    assert got[1][2] >= 1 and got[1][3] == 0 and got[1][5] == 0
    drafts[5, 0] = -1
    assert run(target, None, drafts, u) == oracle.chains(target, None, drafts, u, None, None)


def test_infinite_temperature_is_the_flattest_and_tiny_ones_are_greedy():
    """T = inf weighs every logit above -inf alike, as the largest finite T does; T = NaN is greedy; a T whose 1 / T
    overflows leaves the maximum alone."""
    target, draft, drafts, u = case(4, 3, 700, torch.float32, seed=31)
    target[:, :, ::3] = -math.inf
    t = torch.tensor([math.inf, math.inf, math.nan, 1e-42])
    same = torch.tensor([torch.finfo(torch.float32).max] * 2 + [0.0, 0.0])
    for d in (draft, None):
        assert run(target, d, drafts, u, None, t) == oracle.chains(target, d, drafts, u, None, same)


def test_single_rows_of_any_row_stride():
    """A dimension of one row has no stride of its own."""
    from seedplane_b200 import speculative
    target, _, drafts, u = case(5, 0, 301, torch.float32, seed=33)
    rows = target.cuda().as_strided((5, 1, 301), (301, 1, 1))
    tokens, accepted = speculative.accept_chains(rows, None, drafts.cuda(), u.cuda())
    assert (tokens.tolist(), accepted.tolist()) == oracle.chains(target, None, drafts, u, None, None)
    target, draft, drafts, u = case(5, 1, 301, torch.float32, seed=34)
    tokens, accepted = speculative.accept_chains(target.cuda(), draft.cuda().as_strided((5, 1, 301), (301, 5, 1)), drafts.cuda(), u.cuda())
    assert (tokens.tolist(), accepted.tolist()) == oracle.chains(target, draft, drafts, u, None, None)


def test_identical_distributions_accept_everything_and_extreme_numbers():
    target, _, drafts, u = case(3, 4, 777, torch.float32, seed=11)
    draft = target[:, :4].clone()
    u[:, :4] = 1.0 - 2.0 ** -53
    assert run(target, draft, drafts, u)[1] == [4, 4, 4]
    u[:, 4] = torch.tensor([0.0, 1.0 - 2.0 ** -53, 0.5], dtype=torch.float64)
    got = run(target, draft, drafts, u)
    assert got == oracle.chains(target, draft, drafts, u, None, None)
    assert got[0][0][4] == 0                             # u = 0: the first index with any weight
    # equal rows and a refused draft: nothing is left of p - q, so p itself
    drafts[0, 0] = -1
    assert run(target, draft, drafts, u) == oracle.chains(target, draft, drafts, u, None, None)


@pytest.mark.parametrize("drafter", [True, False])
def test_numbers_next_to_the_border_are_decided_in_64_bits(drafter):
    """u q(x) a millionth under or over p(x), drafts on both sides of it along one chain, and a draw after each."""
    B, n, V = 6, 3, 5000
    target, draft, drafts, u = case(B, n, V, torch.float32, seed=17, spread=1.0, near=0.3)
    if not drafter:
        draft = None
        drafts = target[:, :n].argmax(-1).int()
    temperature = torch.full((B,), 0.7)
    for b in range(B):
        for i in range(n):
            x = int(drafts[b, i])
            dist = lambda row: torch.softmax(row.double() / 0.7, 0)  # noqa: E731
            p, q = float(dist(target[b, i])[x]), float(dist(draft[b, i])[x]) if drafter else 1.0
            u[b, i] = min(p / q, 0.999999) * (1 + (1e-6 if (b >> i) & 1 else -1e-6))
    got = run(target, draft, drafts, u, None, temperature)
    assert got == oracle.chains(target, draft, drafts, u, None, temperature)
    assert set(got[1]) >= {0, 1, 2} if not drafter else True


@pytest.mark.parametrize("drafter", [True, False])
@pytest.mark.parametrize("V", [40, 5000, 50001])
def test_one_number_next_to_the_border(drafter, V):
    """As above for one draft of a chain: accepted ones before it, and behind it all kinds (accepted, refused, a row without
    weight), which follow only if it is accepted."""
    B, n = 24, 3
    target, draft, drafts, u = case(B, n, V, torch.float32, seed=19 + V, spread=1.0, near=0.3)
    u[:, :n] = torch.rand(B, n, generator=torch.Generator().manual_seed(V), dtype=torch.float64)
    if not drafter:
        draft = None
        drafts = target[:, :n].argmax(-1).int()
    near, border = [b % n for b in range(B)], []
    for b in range(B):
        i, x = near[b], int(drafts[b, near[b]])
        dist = lambda row: torch.softmax(row.double() / 0.7, 0)  # noqa: E731
        p, q = float(dist(target[b, i])[x]), float(dist(draft[b, i])[x]) if drafter else 1.0
        border.append(p < 0.99 * q)                      # else any number accepts it
        u[b, :i] = 1e-9                                  # accepted, whatever p and q
        u[b, i] = min(p / q, 0.999999) * (1 + (1e-6 if b // n % 2 else -1e-6))
        if b >= 18:
            target[b, i + 1] = -math.inf                 # behind it: nothing to accept or draw
    temperature = torch.full((B,), 0.7)
    got = run(target, draft, drafts, u, None, temperature)
    assert got == oracle.chains(target, draft, drafts, u, None, temperature)
    assert sum(border) >= 6 and all((got[1][b] > near[b]) == (b // n % 2 == 0) for b in range(B) if border[b])


def test_strided_rows_and_rows_behind_the_counts_are_not_read():
    target, draft, drafts, u = case(3, 3, 999, torch.float32, seed=13)
    counts = torch.tensor([1, 3, 0], dtype=torch.int32)
    want = oracle.chains(target, draft, drafts, u, counts, None)
    wide_t, wide_d = torch.full((3, 5, 1003), math.nan), torch.full((3, 4, 1003), math.nan)
    wide_t[:, :4, 2:1001], wide_d[:, :3, 2:1001] = target, draft
    for b, c in enumerate(counts.tolist()):
        wide_t[b, c + 1:] = math.nan
        wide_d[b, c:] = math.nan
        drafts[b, c:] = 10 ** 6
    from seedplane_b200 import speculative
    t, d = wide_t.cuda()[:, :4, 2:1001], wide_d.cuda()[:, :3, 2:1001]
    tokens, accepted = speculative.accept_chains(t, d, drafts.cuda(), u.cuda(), counts=counts.cuda())
    assert (tokens.tolist(), accepted.tolist()) == want


def test_agrees_with_the_tree_verification_of_one_chain():
    """The distribution of the first emitted token is the target's, drafted or not (100,000 trials of one batch row)."""
    V, trials = 6, 100_000
    g = torch.Generator().manual_seed(3)
    logits, dlogits = torch.randn(V, generator=g), torch.randn(V, generator=g)
    q = torch.softmax(dlogits.double(), 0)
    drafts = torch.multinomial(q, trials, replacement=True, generator=g).int()[:, None]
    u = torch.rand(trials, 2, generator=g, dtype=torch.float64)
    tokens, _ = run(logits.expand(trials, 2, V).contiguous(), dlogits.expand(trials, 1, V).contiguous(), drafts, u)
    first = torch.tensor([t[0] for t in tokens])
    share = torch.bincount(first, minlength=V).double() / trials
    p = torch.softmax(logits.double(), 0)
    # a share's standard deviation is at most sqrt(p (1 - p) / trials): six of them
    assert ((share - p).abs() <= 6 * (p * (1 - p) / trials).sqrt()).all()


def test_captures_into_a_graph():
    from seedplane_b200 import speculative
    target, draft, drafts, u = (t.cuda() for t in case(4, 3, 5000, torch.float32, seed=21))
    out = (torch.zeros(4, 4, dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda"))
    temperature = torch.ones(4, device="cuda")
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        speculative.accept_chains(target, draft, drafts, u, temperature=temperature, out=out)
    for seed in (22, 23):
        for t, new in zip((target, draft, drafts, u), case(4, 3, 5000, torch.float32, seed=seed)):
            t.copy_(new)
        g.replay()
        torch.cuda.synchronize()
        want = oracle.chains(target.cpu(), draft.cpu(), drafts.cpu(), u.cpu(), None, None)
        assert (out[0].tolist(), out[1].tolist()) == want
