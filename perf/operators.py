"""The serving operators of a batch that shares a long prompt prefix: what is timed, and what it has to give.

Three operators, each in its plain form (torch, 32 bits or more) and through the framework's entry points:

* append: a pass's fused q | k | v rows get their bias and position rotation; q goes out, k and v into
  the requests' pages (`seedplane_b200.paged.append`);
* attention: the queries of all requests over the shared prefix's pages and each request's own pages
  (`seedplane_b200.paged.attention`);
* accept: drafted tokens verified against the target's and the drafter's distributions with given
  random numbers (`seedplane_b200.speculative.accept_chains`).

Head counts are those of the repository's Qwen2 configurations: 14 / 2 heads of 64 (0.5B), 12 / 2 of 128
(1.5B), 28 / 4 of 128 (7B), vocabularies of 151,936 and 152,064.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HEADS = {"0.5b": (14, 2, 64), "1.5b": (12, 2, 128), "7b": (28, 4, 128)}
THETA = 1e6


def listed():
    return [
        # one decode step of one request: the smallest call, all latency
        {"name": "append-1tok-0.5b", "op": "append", "heads": "0.5b", "batch": 1, "q_lo": 1, "q_hi": 1, "own_lo": 37, "own_hi": 37,
         "prefix": 512, "page": 16, "dtype": "f32", "rot": 64, "interleaved": False, "bias": True},
        # one decode step of a full batch, fp32 rows as the framework's projections give them
        {"name": "append-64req-7b", "op": "append", "heads": "7b", "batch": 64, "q_lo": 1, "q_hi": 1, "own_lo": 3, "own_hi": 700,
         "prefix": 8192, "page": 64, "dtype": "f32", "rot": 128, "interleaved": False, "bias": True},
        # the packed prompts of a burst, rotated in part and pairwise, bf16 rows without bias
        {"name": "append-prompts-7b-bf16", "op": "append", "heads": "7b", "batch": 23, "q_lo": 17, "q_hi": 700, "own_lo": 700, "own_hi": 1200,
         "prefix": 1024, "page": 128, "dtype": "bf16", "rot": 64, "interleaved": True, "bias": False},
        # a small batch after a short system prompt
        {"name": "attn-4req-0.5b", "op": "attention", "heads": "0.5b", "batch": 4, "q_lo": 1, "q_hi": 1, "own_lo": 1, "own_hi": 90,
         "prefix": 512, "page": 16, "dtype": "f16"},
        # the framework's own precision: fp32 queries over an fp16 cache
        {"name": "attn-16req-1.5b-f32", "op": "attention", "heads": "1.5b", "batch": 16, "q_lo": 1, "q_hi": 1, "own_lo": 20, "own_hi": 600,
         "prefix": 4096, "page": 64, "dtype": "f32"},
        # a full decode batch after a long shared prompt
        {"name": "attn-64req-7b", "op": "attention", "heads": "7b", "batch": 64, "q_lo": 1, "q_hi": 1, "own_lo": 16, "own_hi": 1000,
         "prefix": 8192, "page": 64, "dtype": "f16"},
        # the same batch verifying up to four drafted tokens a request
        {"name": "attn-drafts-7b-bf16", "op": "attention", "heads": "7b", "batch": 48, "q_lo": 1, "q_hi": 5, "own_lo": 33, "own_hi": 777,
         "prefix": 8000, "page": 32, "dtype": "bf16"},
        # questions on one very long document
        {"name": "attn-128req-7b-64k", "op": "attention", "heads": "7b", "batch": 128, "q_lo": 1, "q_hi": 1, "own_lo": 40, "own_hi": 500,
         "prefix": 65536, "page": 128, "dtype": "bf16"},
        # prompts of many tokens after a shared system prompt
        {"name": "attn-prompts-7b", "op": "attention", "heads": "7b", "batch": 12, "q_lo": 60, "q_hi": 512, "own_lo": 512, "own_hi": 640,
         "prefix": 3001, "page": 64, "dtype": "f16"},
        # one request's four drafts: latency
        {"name": "accept-1x4", "op": "accept", "batch": 1, "drafts": 4, "vocab": 151936, "dtype": "f32", "drafter": True, "spread": 3.0},
        # a serving batch with a drafter
        {"name": "accept-32x5", "op": "accept", "batch": 32, "drafts": 5, "vocab": 152064, "dtype": "f32", "drafter": True, "spread": 3.0},
        # drafts looked up in the prompt: no drafter distribution, ragged counts
        {"name": "accept-48x8-lookup", "op": "accept", "batch": 48, "drafts": 8, "vocab": 151936, "dtype": "bf16", "drafter": False, "spread": 4.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("append", "attention", "attention", "accept"))
    if op == "accept":
        drafter = rng.random() < 0.6
        return {"op": op, "batch": _log(rng, 1, 32), "drafts": rng.randint(1, 8 if not drafter else 5),
                "vocab": rng.choice((151936, 152064, _log(rng, 1000, 150000))), "dtype": rng.choice(("f32", "f32", "f16", "bf16")),
                "drafter": drafter, "spread": round(rng.uniform(1.0, 5.0), 2)}
    heads = rng.choice(sorted(HEADS))
    dtype = rng.choice(("f32", "f16", "bf16"))
    page = rng.choice((16, 32, 64, 128, 256))
    if rng.random() < 0.25:                    # packed prompts
        q_lo, q_hi = 1, _log(rng, 8, 400)
        batch = rng.randint(1, 10)
        own_lo, prefix = q_hi, _log(rng, 16, 2500)
    else:                                      # decode steps and short drafts
        q_lo, q_hi = 1, rng.choice((1, 1, 1, 4, 6))
        batch = _log(rng, 1, 64)
        own_lo, prefix = q_hi, _log(rng, 64, 32768)
    own_hi = own_lo + _log(rng, 1, 900)
    case = {"op": op, "heads": heads, "batch": batch, "q_lo": q_lo, "q_hi": q_hi, "own_lo": own_lo, "own_hi": own_hi,
            "prefix": prefix, "page": page, "dtype": dtype}
    if op == "append":
        hd = HEADS[heads][2]
        case |= {"rot": rng.choice((hd, hd, hd // 2)), "interleaved": rng.random() < 0.4, "bias": rng.random() < 0.5}
    return case


def _lens(case):
    """The requests' token counts and own lengths (these tokens among them): a property of the case, not of the seed."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    q = [rng.randint(case["q_lo"], case["q_hi"]) for _ in range(case["batch"])]
    n = [max(rng.randint(case["own_lo"], case["own_hi"]), a) for a in q]
    return q, n


def _pages(case):
    q, n = _lens(case)
    page = case["page"]
    prefix = -(-case["prefix"] // page)
    each = [-(-a // page) for a in n]
    return q, n, prefix, each, prefix + sum(each) + 3


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(int(seed))
    return _prepare_accept(case, g) if case["op"] == "accept" else _prepare_paged(case, g, int(seed))


def _prepare_paged(case, g, seed):
    nh, nkv, hd = HEADS[case["heads"]]
    q_len, own_len, n_prefix, each, n_pages = _pages(case)
    dt = DTYPES[case["dtype"]]
    cache = torch.bfloat16 if dt == torch.bfloat16 else torch.float16
    order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed)).int()
    tables = torch.zeros(len(q_len), max(each), dtype=torch.int32)
    at = n_prefix
    for b, m in enumerate(each):
        tables[b, :m] = order[at:at + m]
        at += m
    shape = (n_pages, nkv, case["page"], hd)
    s = {
        "case": case, "nh": nh, "nkv": nkv, "hd": hd, "prefix": case["prefix"], "max_q": max(q_len), "max_own": max(own_len), "tokens": sum(q_len),
        "k": torch.randn(shape, device="cuda", generator=g, dtype=torch.float32).to(cache),
        "v": torch.randn(shape, device="cuda", generator=g, dtype=torch.float32).to(cache),
        "prefix_table": order[:n_prefix].cuda(), "tables": tables.cuda(),
        "lens": torch.tensor(own_len, dtype=torch.int32, device="cuda"),
        "q_start": torch.tensor([0] + q_len, dtype=torch.int32).cumsum(0).int().cuda(),
    }
    t = s["tokens"]
    if case["op"] == "append":
        s["qkv"] = torch.randn(t, (nh + 2 * nkv) * hd, device="cuda", generator=g, dtype=torch.float32).to(dt)
        s["bias"] = torch.randn((nh + 2 * nkv) * hd, device="cuda", generator=g) if case["bias"] else None
        s["rope"] = _rope(case["prefix"] + s["max_own"], case["rot"]).float().cuda()
        s["q"] = torch.empty(t, nh, hd, device="cuda", dtype=dt)
    else:
        # scores of a spread of about two after the scale, as trained heads have
        s["q"] = (2 * torch.randn(t, nh, hd, device="cuda", generator=g, dtype=torch.float32)).to(dt)
        s["out"] = torch.empty_like(s["q"])
    if own:
        from seedplane_b200 import paged
        s["pages"] = paged.PagedKV.wrap(s["k"], s["v"])
        s["batch"] = paged.PageBatch(s["tables"], s["lens"], q_start=s["q_start"], tokens=t, max_q=s["max_q"],
                                     prefix_table=s["prefix_table"], prefix_len=case["prefix"])
    return s


def _rope(positions, rot):
    """(cos, sin) of every position and rotated pair, in 64 bits."""
    inv = THETA ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    a = torch.arange(positions, dtype=torch.float64)[:, None] * inv
    return torch.stack((a.cos(), a.sin()), -1)


def _prepare_accept(case, g):
    b, n, v = case["batch"], case["drafts"], case["vocab"]
    dt = DTYPES[case["dtype"]]
    target = (case["spread"] * torch.randn(b, n + 1, v, device="cuda", generator=g)).to(dt)
    noise = lambda: torch.rand(b, n, v, device="cuda", generator=g).clamp_(min=1e-30).log_().neg_().log_().neg_()  # noqa: E731
    if case["drafter"]:                        # a drafter that is near the target; its tokens drawn from it
        draft = (target[:, :n].float() + 0.4 * torch.randn(b, n, v, device="cuda", generator=g)).to(dt)
        tokens = (draft.float() + noise()).argmax(-1).int()
        counts = None
    else:                                      # looked up: right often, and fewer than n for some requests
        draft = None
        tokens = target[:, :n].float().argmax(-1).int()
        wrong = torch.rand(b, n, device="cuda", generator=g) < 0.2
        tokens = torch.where(wrong, torch.randint(0, v, (b, n), device="cuda", generator=g, dtype=torch.int32), tokens)
        target.scatter_(2, target[:, :n].float().argmax(-1, keepdim=True), case["spread"] * 4.6 + 2)
        counts = torch.randint(0, n + 1, (b,), device="cuda", generator=g, dtype=torch.int32)
    temperature = 0.6 + 0.5 * torch.rand(b, device="cuda", generator=g)
    u = torch.rand(b, n + 1, device="cuda", generator=g, dtype=torch.float64)
    return {"case": case, "target": target, "draft": draft, "tokens": tokens, "counts": counts, "temperature": temperature, "u": u}


def run(s):
    op = s["case"]["op"]
    if own:
        if op == "append":
            from seedplane_b200 import paged
            paged.append(s["pages"], 0, s["batch"], s["qkv"], s["nh"], s["rope"], bias=s["bias"], interleaved=s["case"]["interleaved"],
                         q_out=s["q"])
            return {"q": s["q"], "k": s["k"], "v": s["v"]}
        if op == "attention":
            from seedplane_b200 import paged
            return paged.attention(s["pages"], 0, s["batch"], s["q"], out=s["out"])
        from seedplane_b200 import speculative
        tokens, accepted = speculative.accept_chains(s["target"], s["draft"], s["tokens"], s["u"], counts=s["counts"],
                                                     temperature=s["temperature"])
        return {"tokens": tokens, "accepted": accepted}
    return {"append": _plain_append, "attention": _plain_attention, "accept": _plain_accept}[op](s)


def _owner(s):
    """Each token's request, and its place among the request's own keys."""
    start = s["q_start"].long()
    t = torch.arange(s["tokens"], device="cuda")
    b = torch.bucketize(t, start[1:], right=True)
    return b, s["lens"].long()[b] - (start[b + 1] - start[b]) + t - start[b]


def _plain_append(s):
    c, nh, nkv, hd = s["case"], s["nh"], s["nkv"], s["hd"]
    x = s["qkv"].float()
    if s["bias"] is not None:
        x = x + s["bias"]
    x = x.view(-1, nh + 2 * nkv, hd)
    b, slot = _owner(s)
    cos, sin = s["rope"][s["prefix"] + slot][:, None].unbind(-1)
    rot = c["rot"]
    head = x[:, :nh + nkv]
    if c["interleaved"]:
        x0, x1 = head[..., 0:rot:2], head[..., 1:rot:2]
        turned = torch.stack((x0 * cos - x1 * sin, x1 * cos + x0 * sin), -1).flatten(-2)
    else:
        x0, x1 = head[..., :rot // 2], head[..., rot // 2:rot]
        turned = torch.cat((x0 * cos - x1 * sin, x1 * cos + x0 * sin), -1)
    head = torch.cat((turned, head[..., rot:]), -1)
    page, place = s["tables"][b, slot // c["page"]].long(), slot % c["page"]
    s["k"][page, :, place] = head[:, nh:].to(s["k"].dtype)
    s["v"][page, :, place] = x[:, nh + nkv:].to(s["v"].dtype)
    s["q"].copy_(head[:, :nh])
    return {"q": s["q"], "k": s["k"], "v": s["v"]}


def _plain_attention(s):
    c, nh, nkv, hd = s["case"], s["nh"], s["nkv"], s["hd"]
    group, nb, mq, n, p = nh // nkv, c["batch"], s["max_q"], s["max_own"], s["prefix"]
    start = s["q_start"].long()
    rows = start[:-1, None] + torch.arange(mq, device="cuda")
    live = rows < start[1:, None]
    q = s["q"].float()[rows.clamp(max=s["tokens"] - 1)]                        # [b, mq, nh, hd]
    q = q.view(nb, mq, nkv, group, hd).permute(0, 2, 1, 3, 4).reshape(nb, nkv, mq * group, hd) / math.sqrt(hd)
    shared = [x[s["prefix_table"].long()].transpose(0, 1).reshape(nkv, -1, hd)[:, :p].float() for x in (s["k"], s["v"])]
    mine = [x[s["tables"].long()].transpose(1, 2).reshape(nb, nkv, -1, hd)[:, :, :n].float() for x in (s["k"], s["v"])]
    a = torch.matmul(q.transpose(0, 1).reshape(nkv, -1, hd), shared[0].transpose(1, 2))   # [nkv, b mq group, p]
    z = torch.matmul(q, mine[0].transpose(2, 3))                               # [b, nkv, mq group, n]
    place = (s["lens"].long() - (start[1:] - start[:-1]))[:, None] + torch.arange(mq, device="cuda")
    seen = torch.arange(n, device="cuda") <= place[:, :, None]                 # [b, mq, n]
    z = z.masked_fill(~seen.repeat_interleave(group, 1)[:, None], -math.inf)
    top_a = a.amax(-1).view(nkv, nb, -1).transpose(0, 1)
    top = torch.maximum(top_a, z.amax(-1))
    a = (a - top.transpose(0, 1).reshape(nkv, -1, 1)).exp_()
    z = (z - top[..., None]).exp_()
    total = a.sum(-1).view(nkv, nb, -1).transpose(0, 1) + z.sum(-1)
    o = torch.matmul(a, shared[1]).view(nkv, nb, -1, hd).transpose(0, 1) + torch.matmul(z, mine[1])
    o = (o / total[..., None]).view(nb, nkv, mq, group, hd).permute(0, 2, 1, 3, 4).reshape(nb, mq, nh, hd)
    return o[live].to(s["q"].dtype)


def _plain_accept(s):
    """In 64 bits: the draw compares a sum of up to 152,064 probabilities with a given number."""
    c, x = s["case"], s["tokens"].long()
    nb, n = x.shape
    warm = s["temperature"].double()[:, None, None]
    p = s["target"].double() / warm
    p = (p - p.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    counts = torch.full((nb,), n, device="cuda") if s["counts"] is None else s["counts"].long()
    if s["draft"] is not None:
        q = s["draft"].double() / warm
        q = (q - q.amax(-1, keepdim=True)).exp()
        q = q / q.sum(-1, keepdim=True)
    else:
        q = torch.zeros_like(p[:, :n]).scatter_(2, x[..., None], 1.0)
    px, qx = p[:, :n].gather(2, x[..., None])[..., 0], q.gather(2, x[..., None])[..., 0]
    i = torch.arange(n, device="cuda")
    good = (s["u"][:, :n] * qx < px) & (i < counts[:, None])
    accepted = good.long().cumprod(1).sum(1)
    b = torch.arange(nb, device="cuda")
    r = p[b, accepted]
    full = accepted == counts
    left = (r - q[b, accepted.clamp(max=n - 1)]).clamp(min=0)
    left = torch.where(full[:, None] | (left.sum(-1, keepdim=True) == 0), r, left)
    run_sum = left.cumsum(-1)
    pick = (run_sum > s["u"][:, n:] * run_sum[:, -1:]).int().argmax(-1)
    tokens = torch.where(i < accepted[:, None], x, -1)
    tokens = torch.cat((tokens, torch.full_like(tokens[:, :1], -1)), 1).scatter_(1, accepted[:, None], pick[:, None])
    return {"tokens": tokens.int(), "accepted": accepted.int()}


def work(case):
    if case["op"] == "accept":
        size = DTYPES[case["dtype"]].itemsize
        rows = case["batch"] * (2 * case["drafts"] + 1 if case["drafter"] else case["drafts"] + 1)
        return {"bytes": rows * case["vocab"] * size + case["batch"] * (case["drafts"] + 1) * 16, "flops": 0}
    nh, nkv, hd = HEADS[case["heads"]]
    q, n, _, each, _ = _pages(case)
    t, size = sum(q), DTYPES[case["dtype"]].itemsize
    if case["op"] == "append":
        return {"bytes": t * ((nh + 2 * nkv) * hd * size + nh * hd * size + 2 * nkv * hd * 2 + case["rot"] * 4 + 4), "flops": 3 * t * (nh + nkv) * case["rot"]}
    keys = case["prefix"] + sum(n)
    seen = sum(a * case["prefix"] + a * m - a * (a - 1) // 2 for a, m in zip(q, n))
    return {"bytes": keys * nkv * hd * 2 * 2 + 2 * t * nh * hd * size + 4 * (sum(each) + case["batch"]), "flops": 4 * seen * nh * hd}


def exact(case, seed):
    """From the definitions in 64 bits, a request at a time. Tokens are whole numbers: no value for them here."""
    if case["op"] == "accept":
        return None
    s = prepare(case, seed)
    nh, nkv, hd, page, p = s["nh"], s["nkv"], s["hd"], case["page"], case["prefix"]
    start, lens, tables = s["q_start"].tolist(), s["lens"].tolist(), s["tables"].long()
    if case["op"] == "append":
        k, v = s["k"].double(), s["v"].double()
        q = torch.empty(s["tokens"], nh, hd, dtype=torch.float64, device="cuda")
        half = case["rot"] // 2
        turn = torch.view_as_complex(s["rope"].double().contiguous())
        for b in range(case["batch"]):
            lo, hi = start[b], start[b + 1]
            x = s["qkv"][lo:hi].double()
            if s["bias"] is not None:
                x = x + s["bias"].double()
            x = x.view(hi - lo, -1, hd)
            slots = torch.arange(lens[b] - (hi - lo), lens[b], device="cuda")
            pairs = torch.arange(half, device="cuda")
            first, second = (2 * pairs, 2 * pairs + 1) if case["interleaved"] else (pairs, pairs + half)
            y = x.clone()
            w = torch.complex(x[:, :nh + nkv, first], x[:, :nh + nkv, second]) * turn[p + slots][:, None]
            y[:, :nh + nkv, first], y[:, :nh + nkv, second] = w.real, w.imag
            q[lo:hi] = y[:, :nh]
            k[tables[b, slots // page], :, slots % page] = y[:, nh:nh + nkv]
            v[tables[b, slots // page], :, slots % page] = y[:, nh + nkv:]
        return {"q": q, "k": k, "v": v}
    out = torch.empty(s["tokens"], nh, hd, dtype=torch.float64, device="cuda")
    for b in range(case["batch"]):
        lo, hi = start[b], start[b + 1]
        at = torch.cat((s["prefix_table"].long().repeat_interleave(page)[:p] * page + torch.arange(p, device="cuda") % page,
                        tables[b].repeat_interleave(page)[:lens[b]] * page + torch.arange(lens[b], device="cuda") % page))
        last = p + lens[b] - (hi - lo) + torch.arange(hi - lo, device="cuda")   # the last key each query sees
        hidden = torch.arange(len(at), device="cuda") > last[:, None]
        for h in range(nkv):
            heads = slice(h * nh // nkv, (h + 1) * nh // nkv)
            kk, vv = (x[at // page, h, at % page].double() for x in (s["k"], s["v"]))
            w = torch.einsum("thd,nd->htn", s["q"][lo:hi, heads].double(), kk) * hd ** -0.5
            w = torch.softmax(w.masked_fill_(hidden, -math.inf), -1)
            out[lo:hi, heads] = torch.einsum("htn,nd->thd", w, vv)
    return out
