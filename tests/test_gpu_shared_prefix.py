"""Passes over pages on the GPU (`sp_forward_pages`, `sp_decode_pages`, `batch.generate_shared`): requests
that share a prefix get the oracle's greedy tokens for prefix + prompt, whatever the lengths, page sizes and
packing; the logits are the contiguous pass's; bad arguments are refused."""
import pytest
import torch

from oracle.qwen_oracle import OracleQwen2
from seedplane_b200.config import PRESETS
from seedplane_b200.randinit import TEST_INIT, make_weights, random_prompt

pytestmark = pytest.mark.gpu


def engine_of(model, **kw):
    from seedplane_b200.engine import CudaQwen2
    cfg = PRESETS[model]
    w = make_weights(cfg, seed=0, dtype=torch.float16, **TEST_INIT)
    return CudaQwen2(cfg, w, **kw), cfg, w


def check_greedy(oracle, ids, got, limit):
    """The oracle's greedy tokens. The engine's logits are held to 1e-3 of the largest |logit| (the test of the
    logits below), so two of them can change places only where the oracle's differ by at most twice that; behind
    such a tie the sequences have nothing in common."""
    want = oracle.greedy(ids, limit)[0]
    assert len(got) == limit
    for i, (g, w) in enumerate(zip(got, want)):
        if g != w:
            row = oracle.prefix_logits(ids + want[:i])
            assert float(row[w] - row[g]) <= 2e-3 * float(row.abs().max()), (i, g, w)
            return


@pytest.fixture(scope="module")
def tiny():
    eng, cfg, w = engine_of("tiny-hd64")
    yield eng, cfg, w
    eng.close()


@pytest.mark.parametrize("model", ["tiny-hd64", "tiny-hd128", "tiny-untied"])
@pytest.mark.parametrize("prefix,page", [(0, 16), (1, 16), (37, 16), (128, 64), (150, 32)])
def test_shared_prefix_matches_the_oracle(model, prefix, page):
    from seedplane_b200.batch import generate_shared
    eng, cfg, w = engine_of(model)
    try:
        oracle = OracleQwen2(cfg, w, kv_fp16=True)
        head = random_prompt(cfg.vocab, prefix, seed=3) if prefix else []
        prompts = [random_prompt(cfg.vocab, n, seed=10 + i) for i, n in enumerate((1, 5, 12, 33, 7, 2))]
        limits = [12, 1, 7, 12, 3, 9]
        got = generate_shared(eng, head, prompts, limits, page_size=page, block=5)
        for p, g, m in zip(prompts, got, limits):
            check_greedy(oracle, list(head) + list(p), g, m)
    finally:
        eng.close()


def test_same_tokens_as_separate_caches_packed_long_and_stopped(tiny):
    from seedplane_b200.batch import MAX_BATCH, generate_batch, generate_shared
    eng, cfg, _ = tiny
    head = random_prompt(cfg.vocab, 90, seed=5)
    prompts = [random_prompt(cfg.vocab, 1 + (29 * i) % 97, seed=50 + i) for i in range(MAX_BATCH + 5)]   # several passes
    full = generate_batch(eng, [list(head) + list(p) for p in prompts], 6)
    assert generate_shared(eng, head, prompts, 6, block=4) == full
    stop = {full[2][2], full[7][4]}
    got = generate_shared(eng, head, prompts, 6, stop=stop, block=3)
    for f, g in zip(full, got):
        cut = next((i for i, t in enumerate(f) if t in stop), None)
        assert g == (f if cut is None else f[:cut + 1])


def test_a_prompt_of_more_than_one_pass(tiny):
    from seedplane_b200.batch import generate_batch, generate_shared
    eng, cfg, _ = tiny
    n = min(700, cfg.max_positions - 80)
    head, prompts = random_prompt(cfg.vocab, 33, seed=6), [random_prompt(cfg.vocab, n, seed=7), random_prompt(cfg.vocab, 9, seed=8)]
    assert generate_shared(eng, head, prompts, 4) == generate_batch(eng, [list(head) + list(p) for p in prompts], 4)


def test_logits_of_a_paged_pass_are_the_contiguous_pass_s(tiny):
    from seedplane_b200.paged import PageBatch
    eng, cfg, _ = tiny
    ids = random_prompt(cfg.vocab, 60, seed=9)
    kv = eng.new_kv(64)
    want, am = eng.forward(kv, list(ids), last_only=True)
    pages = eng.new_pages(5, 16)
    dev = eng.device
    t = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    eng.forward_pages(pages, PageBatch(t([[3, 1]]), t([21]), max_q=21), t(list(ids[:21])))
    argmax, logits = eng.forward_pages(pages, PageBatch(t([[4, 0, 2]]), t([39]), max_q=39, prefix_table=t([3, 1]), prefix_len=21),
                                       t(list(ids[21:])), want_logits=True)
    eng.status()
    kv.close()
    assert int(argmax[0]) == int(am[-1])
    assert float((logits[0] - want[-1]).abs().max() / want[-1].abs().max()) < 1e-3


def test_bad_tables_and_arguments(tiny):
    from seedplane_b200._native import EngineError
    from seedplane_b200.batch import generate_shared
    from seedplane_b200.paged import PageBatch, PagedKV
    eng, cfg, _ = tiny
    dev = eng.device
    t = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    pages = eng.new_pages(2, 16)
    tok = t([1, 2, 3])
    eng.forward_pages(pages, PageBatch(t([[9]]), t([3]), max_q=3), tok)      # a page that does not exist
    with pytest.raises(EngineError):
        eng.status()
    eng.status()
    eng.forward_pages(pages, PageBatch(t([[0]]), t([3]), max_q=3), t([1, cfg.vocab, 3]))
    with pytest.raises(EngineError):
        eng.status()
    eng.status()
    with pytest.raises(ValueError):
        eng.forward_pages(pages, PageBatch(t([[0]]), t([3]), max_q=3), tok[:2])
    with pytest.raises(ValueError):
        eng.forward_pages(PagedKV(cfg.layers + 1, cfg.kv_heads, cfg.head_dim, 2, 16), PageBatch(t([[0]]), t([3]), max_q=3), tok)
    with pytest.raises(ValueError):
        eng.forward_pages(PagedKV(cfg.layers, cfg.kv_heads, cfg.head_dim, 2, 16, torch.bfloat16),
                          PageBatch(t([[0]]), t([3]), max_q=3), tok)
    with pytest.raises(ValueError):
        eng.forward_pages(pages, PageBatch(t([[0]]), t([600]), max_q=600), torch.zeros(600, dtype=torch.int32, device=dev))
    with pytest.raises(ValueError):
        eng.decode_pages(pages, PageBatch(t([[0]]), t([3]), max_q=3), tok, 1)
    with pytest.raises(ValueError):
        eng.decode_pages(pages, PageBatch(t([[0]]), t([3])), tok[:1].clone(), 0)
    with pytest.raises(ValueError):
        generate_shared(eng, [1], [[]], 3)
    with pytest.raises(ValueError):
        generate_shared(eng, [1], [[2]], cfg.max_positions)
    assert generate_shared(eng, [1], [], 3) == []


def test_grouped_lease_with_a_prefix(tiny):
    from seedplane_b200.hive.agent import GreedyExecutor
    eng, cfg, _ = tiny
    head = [int(v) for v in random_prompt(cfg.vocab, 20, seed=30)]
    tails = [[int(v) for v in random_prompt(cfg.vocab, n, seed=31 + n)] for n in (3, 8, 1)]
    ex = GreedyExecutor(eng, 64)
    plain = ex({"batch": [{"ids": head + p, "max_new_tokens": 5} for p in tails]})
    shared = ex({"prefix_ids": head, "batch": [{"ids": p, "max_new_tokens": 5} for p in tails]})
    assert plain == shared
    with pytest.raises(ValueError):
        ex({"prefix_ids": head, "batch": [{"ids": tails[0], "max_new_tokens": 60}]})


def test_passes_are_not_captured(tiny):
    """The engine may move its workspace for a later, larger pass: a graph must not keep it."""
    from seedplane_b200.paged import PageBatch
    eng, cfg, _ = tiny
    dev = eng.device
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    pages = eng.new_pages(4, 64)
    batch, tokens = PageBatch(i32([[0], [1]]), i32([1, 1])), i32([3, 4])
    want = eng.forward_pages(pages, batch, tokens)[0].tolist()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        for call in (lambda: eng.forward_pages(pages, batch, tokens), lambda: eng.decode_pages(pages, batch, tokens, 2)):
            with pytest.raises(RuntimeError, match="captured"):
                call()
    assert eng.forward_pages(pages, batch, tokens)[0].tolist() == want
    eng.status()
