"""`batch.generate_shared` on the CPU with an engine that keeps token ids in its pages and answers a function of every
id a row sees: the packing, the tables, and groups of requests that take one another's pages."""
import types

import pytest
import torch

from seedplane_b200.batch import MAX_BATCH, generate_shared
from seedplane_b200.hive.agent import GreedyExecutor

VOCAB = 997


def next_token(ids):
    h = 7
    for t in ids:
        h = (h * 31 + t + 1) % VOCAB
    return h


class PageEngine:
    device = torch.device("cpu")
    cfg = types.SimpleNamespace(max_positions=4000)

    def new_kv(self, capacity):
        return types.SimpleNamespace(capacity=capacity, length=0)

    def new_pages(self, n_pages, page_size):
        self.n_pages, self.page, self.passes = n_pages, page_size, 0
        self.ids = [[None] * page_size for _ in range(n_pages)]
        return self

    def _seen(self, batch, b, n):
        keys = [self.ids[int(batch.prefix_table[j // self.page])][j % self.page] for j in range(batch.prefix_len)]
        return keys + [self.ids[int(batch.tables[b, j // self.page])][j % self.page] for j in range(n)]

    def forward_pages(self, pages, batch, tokens):
        self.passes += 1
        assert 1 <= batch.batch <= 256 and batch.tokens <= 512
        starts = batch.q_start.tolist() if batch.q_start is not None else [b * batch.max_q for b in range(batch.batch + 1)]
        assert starts[-1] == batch.tokens == len(tokens)
        out = []
        for b in range(batch.batch):
            n, q = int(batch.lens[b]), starts[b + 1] - starts[b]
            assert 1 <= q <= batch.max_q and n <= batch.tables.shape[1] * self.page
            for i in range(q):
                key = n - q + i
                self.ids[int(batch.tables[b, key // self.page])][key % self.page] = int(tokens[starts[b] + i])
        for b in range(batch.batch):
            out.append(next_token(self._seen(batch, b, int(batch.lens[b]))))
        return torch.tensor(out, dtype=torch.int32), None

    def decode_pages(self, pages, batch, tokens, n_steps):
        rows = []
        for _ in range(n_steps):
            batch.lens += 1
            tokens, _ = self.forward_pages(pages, batch, tokens)
            rows.append(tokens)
        return torch.stack(rows)

    def status(self):
        pass


def expected(prefix, prompts, limits, stop=()):
    out = []
    for p, m in zip(prompts, limits):
        ids, got = list(prefix) + list(p), []
        while len(got) < m and not (got and got[-1] in stop):
            got.append(next_token(ids + got))
        out.append(got)
    return out


@pytest.mark.parametrize("group", [None, 1, 3, 64, 1000])
@pytest.mark.parametrize("prefix,page", [(0, 16), (37, 16), (700, 64)])
def test_groups_give_the_same_tokens(group, prefix, page):
    eng = PageEngine()
    head = [(5 * i) % VOCAB for i in range(prefix)]
    prompts = [[(i * 13 + j) % VOCAB for j in range(1 + (29 * i) % 97)] for i in range(20)] + [[1] * 600]
    limits = [1 + (7 * i) % 11 for i in range(21)]
    got = generate_shared(eng, head, prompts, limits, block=4, page_size=page, group=group)
    want = expected(head, prompts, limits)
    assert got == want
    need = [-(-(len(p) + m) // page) for p, m in zip(prompts, limits)]
    size = group or 21
    assert eng.n_pages == -(-prefix // page) + max(sum(need[b:b + size]) for b in range(0, 21, size))
    stop = {want[4][0], want[9][2]}
    assert generate_shared(eng, head, prompts, limits, stop=stop, block=4, page_size=page, group=group) == \
        expected(head, prompts, limits, stop)


def test_group_sizes_are_checked():
    with pytest.raises(ValueError):
        generate_shared(PageEngine(), [1], [[2]], 3, group=0)


def test_a_long_lease_holds_the_pages_of_one_group():
    eng = PageEngine()
    ex = GreedyExecutor(eng, 64)
    items = [{"ids": [n, n + 1], "max_new_tokens": 3} for n in range(3 * MAX_BATCH + 5)]
    got = ex({"prefix_ids": list(range(40)), "batch": items})
    assert [r["tokens"] for r in got["batch"]] == expected(range(40), [it["ids"] for it in items], [3] * len(items))
    assert eng.n_pages == 1 + MAX_BATCH
