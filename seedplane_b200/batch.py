"""Runtime request batching: greedy generation of independent requests together on one engine.

The reference decodes one request per native session and its HIVE agents report `batch_size: 1`
(`seedplane/hive/pool.py:465-466`; a batched inference API is listed as not built,
`README.md:68`). Here the requests of a batch share every decode step: `sp_decode_batch` runs ONE
batched pass per step over the batch's tokens, each reading and writing its own KV cache, so the
weights stream from HBM once per step for all of them. Every request's tokens are its own greedy
continuation, the same as decoding it alone.

`generate_batch` packs the requests' prompts into batched passes (`sp_prefill_batch`: every token
writes and reads its own request's cache), then decodes the batch in device blocks (each block's
argmaxes are fed back on the GPU); after a block the host cuts each request at its stop token or
length limit and drops finished requests from the batch.
"""
from __future__ import annotations

from typing import Iterable, List, Optional, Sequence

import torch

MAX_BATCH = 64                          # requests per sp_decode_batch call
MAX_PREFILL_BATCH = 256                 # prompts per sp_prefill_batch call
MAX_PASS_TOKENS = 512                   # rows of a packed pass over pages (sp_forward_pages)


def generate_batch(engine, prompts: Sequence[Sequence[int]], max_new_tokens, stop: Iterable[int] = (),
                   block: int = 16, kvs: Optional[Sequence] = None, timer=None) -> List[List[int]]:
    """Greedy tokens of every prompt (each up to max_new_tokens, ending at the first stop token,
    which is included). `max_new_tokens` is one limit or one per request. `kvs`: caches to use (one
    per request, each with room for its prompt and tokens; their contents are replaced), else new
    ones for this call. `timer(start: bool)` brackets the device work."""
    n_req = len(prompts)
    if n_req == 0:
        return []
    limits = [int(max_new_tokens)] * n_req if isinstance(max_new_tokens, int) else [int(m) for m in max_new_tokens]
    if len(limits) != n_req or any(m < 1 for m in limits):
        raise ValueError("every request needs max_new_tokens >= 1")
    stops = {int(s) for s in stop}
    prompts = [[int(t) for t in p] for p in prompts]
    if any(not p for p in prompts):
        raise ValueError("empty prompt")
    own = kvs is None
    if own:
        kvs = [engine.new_kv(len(p) + m) for p, m in zip(prompts, limits)]
    elif len(kvs) < n_req or any(kv.capacity < len(p) + m for kv, p, m in zip(kvs, prompts, limits)):
        raise ValueError("a request does not fit its cache")
    try:
        if timer:
            timer(True)
        firsts = []
        for kv in kvs[:n_req]:
            kv.length = 0
        for c0 in range(0, n_req, MAX_PREFILL_BATCH):      # the prompts packed into batched passes
            firsts.append(engine.prefill_batch(kvs[c0:c0 + MAX_PREFILL_BATCH], prompts[c0:c0 + MAX_PREFILL_BATCH]))
        out = [[t] for t in torch.cat(firsts).cpu().tolist()]
        done = [o[0] in stops or m == 1 for o, m in zip(out, limits)]
        while True:
            active = [b for b in range(n_req) if not done[b]]
            if not active:
                break
            for c0 in range(0, len(active), MAX_BATCH):
                group = active[c0:c0 + MAX_BATCH]
                n = max(1, min(block, min(limits[b] - len(out[b]) for b in group)))
                toks = engine.decode_batch([kvs[b] for b in group], [out[b][-1] for b in group],
                                           [len(prompts[b]) + len(out[b]) - 1 for b in group], n)
                rows = toks.cpu().tolist()               # [n][len(group)]
                for j, b in enumerate(group):
                    for i in range(n):
                        t = rows[i][j]
                        out[b].append(t)
                        if t in stops or len(out[b]) >= limits[b]:
                            done[b] = True
                            break
        if timer:
            timer(False)
        return out
    finally:
        if own:
            for kv in kvs:
                kv.close()


def generate_shared(engine, prefix: Sequence[int], prompts: Sequence[Sequence[int]], max_new_tokens, stop: Iterable[int] = (),
                    block: int = 16, page_size: int = 64, timer=None, group: Optional[int] = None) -> List[List[int]]:
    """`generate_batch` for requests that all start with `prefix`: the same greedy tokens as for the prompts
    prefix + prompt, with the prefix run through the model once and its keys and values kept once, in pages that every
    request reads (the attention of a step reads them once for the whole batch). Arguments as `generate_batch`; each
    prompt has at least one token. `group`: at most so many requests hold pages at a time (None: all of them); the next
    ones take the pages of those before."""
    n_req = len(prompts)
    if n_req == 0:
        return []
    limits = [int(max_new_tokens)] * n_req if isinstance(max_new_tokens, int) else [int(m) for m in max_new_tokens]
    if len(limits) != n_req or any(m < 1 for m in limits):
        raise ValueError("every request needs max_new_tokens >= 1")
    prefix = [int(t) for t in prefix]
    prompts = [[int(t) for t in p] for p in prompts]
    if any(not p for p in prompts):
        raise ValueError("empty prompt")
    if len(prefix) + max(len(p) + m for p, m in zip(prompts, limits)) > engine.cfg.max_positions:
        raise ValueError("a request exceeds the model's positions")
    if group is not None and group < 1:
        raise ValueError("group must be positive")
    stops = {int(s) for s in stop}
    groups = [slice(b, b + (group or n_req)) for b in range(0, n_req, group or n_req)]
    need = [-(-(len(p) + m) // page_size) for p, m in zip(prompts, limits)]
    n_prefix = -(-len(prefix) // page_size)
    pages = engine.new_pages(n_prefix + max(sum(need[g]) for g in groups), page_size)
    if timer:
        timer(True)
    shared = _run_prefix(engine, pages, prefix, n_prefix)
    out = []
    for g in groups:
        out += _run_group(engine, pages, shared, n_prefix, prompts[g], limits[g], need[g], stops, block)
    if timer:
        timer(False)
    engine.status()
    return out


def _int32(v, dev):
    return torch.tensor(v, dtype=torch.int32).to(dev)


def _run_prefix(engine, pages, prefix, n_prefix) -> dict:
    """The prefix's keys and values into the first pages, as one request's own keys; how a `PageBatch` names them."""
    from .paged import PageBatch
    dev = engine.device
    prefix_table = torch.arange(n_prefix, dtype=torch.int32, device=dev)
    for c0 in range(0, len(prefix), MAX_PASS_TOKENS):
        part = prefix[c0:c0 + MAX_PASS_TOKENS]
        one = PageBatch(prefix_table[None], _int32([c0 + len(part)], dev), max_q=len(part))
        engine.forward_pages(pages, one, _int32(part, dev))
    return dict(prefix_table=prefix_table, prefix_len=len(prefix))


def _run_group(engine, pages, shared, first_page, prompts, limits, need, stops, block) -> List[List[int]]:
    """The requests' tokens after a prefix that has been run; their pages (`need` each) start at `first_page`."""
    from .paged import PageBatch
    n_req, dev = len(prompts), engine.device
    tables = torch.zeros((n_req, max(need)), dtype=torch.int32)
    at = first_page
    for b, m in enumerate(need):
        tables[b, :m] = torch.arange(at, at + m, dtype=torch.int32)
        at += m
    tables = tables.to(dev)
    done_rows, firsts = [0] * n_req, [None] * n_req
    b = 0
    while b < n_req:                                           # prompts packed into passes; a long one in several
        rows, room = [], MAX_PASS_TOKENS
        while b < n_req and room > 0 and len(rows) < MAX_PREFILL_BATCH:
            take = min(room, len(prompts[b]) - done_rows[b])
            rows.append((b, done_rows[b], take))
            done_rows[b] += take
            room -= take
            if done_rows[b] < len(prompts[b]):
                break
            b += 1
        flat = [t for r, r0, take in rows for t in prompts[r][r0:r0 + take]]
        starts = [0]
        for _, _, take in rows:
            starts.append(starts[-1] + take)
        part = PageBatch(tables[rows[0][0]:rows[-1][0] + 1], _int32([r0 + take for _, r0, take in rows], dev), q_start=_int32(starts, dev),
                         tokens=len(flat), max_q=max(take for _, _, take in rows), **shared)
        argmax, _ = engine.forward_pages(pages, part, _int32(flat, dev))
        for j, (r, r0, take) in enumerate(rows):
            if r0 + take == len(prompts[r]):
                firsts[r] = argmax[j]
    out = [[t] for t in torch.stack(firsts).cpu().tolist()]
    done = [o[0] in stops or m == 1 for o, m in zip(out, limits)]
    while not all(done):
        active = [b for b in range(n_req) if not done[b]]
        for c0 in range(0, len(active), MAX_BATCH):
            group = active[c0:c0 + MAX_BATCH]
            n = max(1, min(block, min(limits[b] - len(out[b]) for b in group)))
            step = PageBatch(tables[_int32(group, dev).long()], _int32([len(prompts[b]) + len(out[b]) - 1 for b in group], dev), **shared)
            rows = engine.decode_pages(pages, step, _int32([out[b][-1] for b in group], dev), n).cpu().tolist()
            for j, b in enumerate(group):
                for i in range(n):
                    out[b].append(rows[i][j])
                    if rows[i][j] in stops or len(out[b]) >= limits[b]:
                        done[b] = True
                        break
    return out
