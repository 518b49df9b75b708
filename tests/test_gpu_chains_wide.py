"""`speculative.accept_chains` over vocabularies of millions: a row's fp32 sum is joined from thousands of chunks, and a
draft whose number lies within what those may be off is decided in 64 bits."""
import pytest
import torch

import paged_oracle as oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V", [2_000_003, 20_000_001])
@pytest.mark.parametrize("drafter", [True, False])
def test_drafts_near_the_border(V, drafter):
    from seedplane_b200 import speculative
    g = torch.Generator("cuda").manual_seed(V)
    target = torch.randn(1, 2, V, device="cuda", generator=g)
    draft = target[:, :1] + 0.3 * torch.randn(1, 1, V, device="cuda", generator=g) if drafter else None
    target[0, 0, V // 2] = 18.0                          # a token of some weight
    drafts = torch.tensor([[V // 2]], dtype=torch.int32, device="cuda")
    p = float(torch.softmax(target[0, 0].double(), 0)[V // 2])
    if drafter:
        draft[0, 0, V // 2] = 19.0
    q = float(torch.softmax(draft[0, 0].double(), 0)[V // 2]) if drafter else 1.0
    assert p < 0.98 * q
    for off in (-1e-4, -1e-6, -1e-9, 1e-9, 1e-6, 1e-4):
        u = torch.tensor([[p / q * (1 + off), 0.37]], dtype=torch.float64, device="cuda")
        tokens, accepted = speculative.accept_chains(target, draft, drafts, u)
        assert (tokens.tolist(), accepted.tolist()) == oracle.chains(target, draft, drafts, u, None, None)
        assert accepted.tolist() == [int(off < 0)]
