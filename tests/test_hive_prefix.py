"""`prefix_ids` in every payload a HIVE agent takes: alone, beside a batch, and inside one (CPU, a fake engine)."""
import threading
import types

import pytest
import torch

import seedplane_b200.batch as batch
from seedplane_b200.hive import HiveBroker
from seedplane_b200.hive.agent import GreedyExecutor, native_generate


class FakeEngine:
    """Answers the sum of the ids it was given, then counts up."""
    device = torch.device("cpu")

    def __init__(self):
        self.calls = []

    def new_kv(self, capacity):
        return types.SimpleNamespace(capacity=capacity, length=0)

    def forward(self, kv, ids, want_logits, last_only):
        self.calls.append(ids.tolist())
        return None, torch.tensor([int(ids.sum())])

    def decode(self, kv, first, pos, n):
        return torch.arange(first + 1, first + 1 + n), None


def answers(prompts, limits):
    limits = [limits] * len(prompts) if isinstance(limits, int) else limits
    return [[sum(p) + i for i in range(m)] for p, m in zip(prompts, limits)]


@pytest.fixture
def executor(monkeypatch):
    eng = FakeEngine()
    monkeypatch.setattr(torch.cuda, "set_device", lambda dev: None)

    def plain(engine, prompts, limits, **kw):
        engine.calls.append(("batch", [list(p) for p in prompts]))
        return answers(prompts, limits)

    def shared(engine, prefix, prompts, limits, **kw):
        engine.calls.append(("shared", list(prefix), [list(p) for p in prompts]))
        return answers([list(prefix) + list(p) for p in prompts], limits)

    monkeypatch.setattr(batch, "generate_batch", plain)
    monkeypatch.setattr(batch, "generate_shared", shared)
    return GreedyExecutor(eng, 40)


def tokens(result):
    return [r["tokens"] for r in result["batch"]]


def test_a_single_request_follows_its_prefix(executor):
    got = executor({"ids": [5, 6], "prefix_ids": [1, 2, 3], "max_new_tokens": 3})
    assert executor.engine.calls == [[1, 2, 3, 5, 6]] and got["tokens"] == [17, 18, 19]
    assert executor({"ids": [1, 2, 3, 5, 6], "max_new_tokens": 3}) == got
    assert executor({"ids": [1, 2, 3, 5, 6], "prefix_ids": [], "max_new_tokens": 3}) == got
    with pytest.raises(ValueError):
        executor({"ids": [5], "prefix_ids": list(range(30)), "max_new_tokens": 10})     # 41 of 40
    with pytest.raises(ValueError):
        executor({"ids": [], "prefix_ids": [1]})


def test_a_common_prefix_inside_a_batch_is_shared(executor):
    items = [{"ids": [4], "max_new_tokens": 2}, {"ids": [5, 6], "max_new_tokens": 1}]
    beside = executor({"prefix_ids": [1, 2], "batch": items})
    inside = executor({"batch": [dict(it, prefix_ids=[1, 2]) for it in items]})
    assert beside == inside and tokens(beside) == [[7, 8], [14]]
    assert [c[0] for c in executor.engine.calls] == ["shared", "shared"]


def test_different_prefixes_inside_a_batch(executor):
    got = executor({"batch": [{"ids": [4], "prefix_ids": [1], "max_new_tokens": 1}, {"ids": [5], "max_new_tokens": 1},
                              {"ids": [6], "prefix_ids": [2, 3], "max_new_tokens": 2}]})
    assert executor.engine.calls == [("batch", [[1, 4], [5], [2, 3, 6]])]
    assert tokens(got) == [[5], [5], [11, 12]]
    with pytest.raises(ValueError):
        executor({"batch": [{"ids": [4] * 20, "prefix_ids": [1] * 20, "max_new_tokens": 1}, {"ids": [5]}]})
    with pytest.raises(ValueError):
        executor({"batch": [{"ids": [], "prefix_ids": [1]}, {"ids": [5]}]})


def test_prefixes_beside_and_inside_a_batch_are_refused(executor):
    with pytest.raises(ValueError, match="both"):
        executor({"prefix_ids": [1], "batch": [{"ids": [4], "prefix_ids": [1]}]})
    assert executor.engine.calls == []


def test_grouped_leases_carry_their_prefix(executor):
    """The broker's groups keep each payload whole, so requests with one prefix are run together after it."""
    with HiveBroker(pull_poll_s=0.02) as broker:
        agent = broker.local_agent("gpu0", caps=("generate",), models=("m",), execute=executor)
        t = threading.Thread(target=agent.run, daemon=True)
        t.start()
        futs = broker.submit_batch([{"ids": [n], "prefix_ids": [7, 8], "max_new_tokens": 1} for n in range(3)], model="m",
                                   require_profiles=False, group_per_worker=True)
        assert [f.result(timeout=5)["tokens"] for f in futs] == [[15], [16], [17]]
    t.join(timeout=5)
    assert executor.engine.calls == [("shared", [7, 8], [[0], [1], [2]])]


def test_native_requests_follow_their_prefix():
    class Native:
        last_tokens, last, info = [9], {}, {"device": "x"}

        def generate(self, **kw):
            self.got = kw
            return ["t"]

    eng = Native()
    native_generate(eng, {"ids": [3], "prefix_ids": [1, 2], "max_new_tokens": 4})
    assert eng.got == {"ids": [1, 2, 3], "reset": True, "max_new_tokens": 4}
    native_generate(eng, {"ids": [3]})
    assert eng.got["ids"] == [3]
    with pytest.raises(ValueError):
        native_generate(eng, {"text": "a", "prefix_ids": [1]})


def test_no_prefix_by_any_name(executor):
    plain = executor({"ids": [5, 6], "max_new_tokens": 2})
    assert executor({"ids": [5, 6], "prefix_ids": None, "max_new_tokens": 2}) == plain
    batch_of = {"batch": [{"ids": [4], "prefix_ids": None, "max_new_tokens": 1}], "prefix_ids": None}
    assert tokens(executor(batch_of)) == [[4]]
