"""`speculative.accept_chains` at the ends of its range: temperatures down to the smallest, logits of any finite
size, rows masked by the type's lowest value. The same tokens as the rule on lists in 64 bits."""
import pytest
import torch

import paged_oracle as oracle
from test_gpu_chains import case, run

pytestmark = pytest.mark.gpu

TINY = [1e-6, 1e-9, 1e-12, 1e-13, 1e-15, 1e-18, 1e-20, 1e-21, 1e-25, 1e-30, 1e-38]


@pytest.mark.parametrize("dt", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("V", [40, 5000])
def test_small_temperatures_leave_the_maximum_alone(V, dt):
    """Certain drafts (the target's own maximum) are accepted at every temperature, and every draw is a row's maximum."""
    B = len(TINY)
    temperature = torch.tensor(TINY)
    for n in (0, 3):
        target, draft, drafts, u = case(B, n, V, torch.float32, seed=V + n, spread=5.0)
        # the largest logits 5 to 25, apart by more than a rounding of the type
        top = target.argmax(-1, keepdim=True)
        target.scatter_(2, top, 25.0 + torch.rand(top.shape, generator=torch.Generator().manual_seed(1)))
        target, draft = target.to(dt), draft.to(dt)
        drafts = target[:, :n].argmax(-1).int()
        for d in ((draft, target[:, :n].clone(), None) if n else (None,)):
            got = run(target, d, drafts, u, None, temperature)
            assert got == oracle.chains(target, d, drafts, u, None, temperature)
            assert got[1] == [n] * B and all(row[n] == int(target[b, n].argmax()) for b, row in enumerate(got[0]))
        if n:                                            # and drafts that are not the maximum
            wrong = (drafts + 1) % V
            for d in (draft, None):
                assert run(target, d, wrong, u, None, temperature) == oracle.chains(target, d, wrong, u, None, temperature)


@pytest.mark.parametrize("size", [1e6, 1e12, 1e20, 1e30, 3e37])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_logits_of_any_size(size, dt):
    for n in (0, 2):
        target, draft, drafts, u = case(6, n, 3000, torch.float32, seed=41 + n, spread=1.0)
        target, draft = (target * size).to(dt), (draft * size).to(dt)
        target[3:, :, 2000] = target[3:, :, 1000] = 8 * size     # two maxima share the weight
        certain = target[:, :n].argmax(-1).int()
        for x in (drafts, certain):
            for d in ((draft, None) if n else (None,)):
                # a temperature of the logits' size flattens them
                for t in (None, torch.tensor([1.0, size, size / 4, 1e-3, size, 1.0])):
                    assert run(target, d, x, u, None, t) == oracle.chains(target, d, x, u, None, t)


@pytest.mark.parametrize("dt", [torch.float32, torch.float16, torch.bfloat16])
def test_rows_of_the_types_lowest_value(dt):
    """A row masked everywhere by the lowest value is flat; one masked but for some tokens draws among those."""
    low = torch.finfo(dt).min
    target, draft, drafts, u = case(4, 2, 999, dt, seed=43)
    target[0, :] = low
    draft[1, :] = low
    target[2, :, 7:] = low
    drafts[2, :] = 3
    target[3, 1:] = low
    for d in (draft, None):
        for t in (None, torch.tensor([0.7, 1e-3, 1e-12, 2.0])):
            assert run(target, d, drafts, u, None, t) == oracle.chains(target, d, drafts, u, None, t)
