"""The paged operators in 64 bits, a request at a time, and ragged batches to run them on."""
import math
import random

import torch

F64 = torch.float64


def make_batch(*, q, lens, prefix, page, nkv, hd, dtype, layers=1, seed=0, tail_rows=0, nhd=False, garbage=float("nan")):
    """Random pages (every slot that no key owns holds `garbage`), shuffled tables, and the lists they came from."""
    g = torch.Generator("cuda").manual_seed(seed)
    rng = random.Random(seed)
    each = [-(-n // page) for n in lens]
    n_prefix = -(-prefix // page)
    total = n_prefix + sum(each) + 2
    order = list(range(total))
    rng.shuffle(order)
    prefix_pages, at = order[:n_prefix], n_prefix
    width = max(each + [1])
    tables = torch.full((len(q), width), -7, dtype=torch.int32)     # entries behind a request's pages are not read
    own = []
    for b, m in enumerate(each):
        tables[b, :m] = torch.tensor(order[at:at + m], dtype=torch.int32)
        own.append(order[at:at + m])
        at += m
    shape = (layers, total, page, nkv, hd) if nhd else (layers, total, nkv, page, hd)
    kv = []
    for _ in range(2):
        t = torch.full(shape, garbage, device="cuda", dtype=dtype)
        t = t.transpose(2, 3) if nhd else t
        for pages, n in [(prefix_pages, prefix)] + [(own[b], lens[b]) for b in range(len(q))]:
            for i, p in enumerate(pages):
                m = min(page, n - i * page)
                t[:, p, :, :m] = torch.randn(layers, nkv, m, hd, device="cuda", generator=g).to(dtype)
        kv.append(t)
    start = [0]
    for n in q:
        start.append(start[-1] + n)
    return dict(k=kv[0], v=kv[1], tables=tables.cuda(), lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                q_start=torch.tensor(start, dtype=torch.int32, device="cuda"), start=start, q=q, len=lens, prefix=prefix,
                prefix_table=torch.tensor(prefix_pages, dtype=torch.int32, device="cuda"), prefix_pages=prefix_pages, own=own,
                page=page, rows=start[-1] + tail_rows)


def keys_of(s, b, which, layer=0):
    """K (or V) of every key request b sees, in order: [kv_heads, keys, head_dim] in 64 bits."""
    t = s[which][layer]
    parts = [t[p] for p in s["prefix_pages"]]
    shared = torch.cat(parts, 1)[:, :s["prefix"]] if parts else t[:0].transpose(0, 1).reshape(t.shape[1], 0, t.shape[3])
    parts = [t[p] for p in s["own"][b]]
    mine = torch.cat(parts, 1)[:, :s["len"][b]] if parts else shared[:, :0]
    return torch.cat((shared, mine), 1).to(F64)


def attention(s, q, scale, layer=0):
    """(out, sum of p |v|, largest sum of |q k| scale, log-sum-exp) per row, 64 bits; rows that see nothing: 0, 0, 0, -inf."""
    nh, hd = q.shape[1:]
    out = torch.zeros(s["start"][-1], nh, hd, dtype=F64, device="cuda")
    absum, size = torch.zeros_like(out), torch.zeros(out.shape[:2], dtype=F64, device="cuda")
    lse = torch.full(out.shape[:2], -math.inf, dtype=F64, device="cuda")
    for b, n in enumerate(s["q"]):
        k, v = keys_of(s, b, "k", layer), keys_of(s, b, "v", layer)
        group = nh // k.shape[0]
        for i in range(n):
            t = s["start"][b] + i
            m = s["prefix"] + s["len"][b] - n + i + 1
            if m <= 0:
                continue
            x = q[t].to(F64).view(k.shape[0], group, hd)
            z = torch.einsum("kgd,knd->kgn", x, k[:, :m]) * scale
            p = torch.softmax(z, -1)
            out[t] = torch.einsum("kgn,knd->kgd", p, v[:, :m]).reshape(nh, hd)
            absum[t] = torch.einsum("kgn,knd->kgd", p, v[:, :m].abs()).reshape(nh, hd)
            size[t] = (torch.einsum("kgd,knd->kgn", x.abs(), k[:, :m].abs()) * scale).amax(-1).reshape(nh)
            lse[t] = torch.logsumexp(z, -1).reshape(nh)
    return out, absum, size, lse


def attention_bounds(q_dtype, cache_dtype, hd, keys, absum, size, ref):
    """How far a row's values may be off. The output's rounding: eps / 2 of the value. The probabilities are rounded to the
    cache's type (fp32 queries: to 2^-22, as two halves): that share of sum p |v|. A score is off by at most hd roundings of
    2^-23 of sum |q k| (the tensor cores may truncate; fp32 queries are held to 2^-22 besides), 2^-22 of itself in the scaling
    and 2^-22 in the exponential: a probability by twice that (numerator and sum). Sums over keys: 2^-23 a step of 16 keys,
    and one for each join."""
    split = q_dtype == torch.float32
    p = 2.0 ** -22 if split else torch.finfo(cache_dtype).eps / 2
    score = size * (hd * 2.0 ** -23 + 2.0 ** -22 + (2.0 ** -22 if split else 0)) + 2.0 ** -22
    steps = (keys / 16 + 64) * 2.0 ** -23
    return torch.finfo(q_dtype).eps / 2 * ref.abs() + (p + 2 * score + 2 * steps)[..., None] * absum + 1e-30


def append(s, qkv, bias, rope, positions, nh, rot, interleaved):
    """Rotated q, k and unrotated v rows in 64 bits, and the sizes their roundings go by."""
    nkv, hd = s["k"].shape[2], s["k"].shape[4]
    n = s["start"][-1]
    x = qkv[:n].to(F64)
    if bias is not None:
        x = x + bias.to(F64)
    x = x.reshape(n, nh + 2 * nkv, hd)
    y, size = x.clone(), x.abs()
    for t in range(n):
        c, sn = rope[positions[t], :, 0].to(F64), rope[positions[t], :, 1].to(F64)
        for j in range(rot // 2):
            a, b = (2 * j, 2 * j + 1) if interleaved else (j, j + rot // 2)
            u, w = x[t, :nh + nkv, a], x[t, :nh + nkv, b]
            y[t, :nh + nkv, a], y[t, :nh + nkv, b] = u * c[j] - w * sn[j], w * c[j] + u * sn[j]
            size[t, :nh + nkv, a] = size[t, :nh + nkv, b] = u.abs() + w.abs()
    return y, size


def chains(target, draft, drafts, u, counts, temperature):
    """The verification rule on lists, 64 bits: (tokens, accepted) per request."""
    toks, accs = [], []
    B, n1, V = target.shape
    for b in range(B):
        T = 1.0 if temperature is None else float(temperature[b])
        cnt = n1 - 1 if counts is None else max(0, min(n1 - 1, int(counts[b])))

        def dist(row):
            z = torch.where(torch.isnan(row), torch.full_like(row, -math.inf), row).to(F64)
            m = z.max()
            if m == -math.inf:
                return torch.zeros_like(z)
            e = torch.where(z == m, torch.ones_like(z), torch.exp((z - m) / T) if T > 0 else torch.zeros_like(z))
            if not T > 0:
                e = torch.zeros_like(z)
                e[int((z == m).nonzero()[0])] = 1.0
            return e / e.sum()

        acc = 0
        while acc < cnt:
            p, x = dist(target[b, acc]), int(drafts[b, acc])
            if not 0 <= x < V:
                break
            if not T > 0:
                ok = bool(p[x] == 1.0)
            else:
                q = 1.0 if draft is None else float(dist(draft[b, acc])[x])
                ok = float(u[b, acc]) * q < float(p[x])
            if not ok:
                break
            acc += 1
        p = dist(target[b, acc])
        r = p
        if acc < cnt and T > 0:
            if draft is None:
                q = torch.zeros_like(p)
                if 0 <= int(drafts[b, acc]) < V:
                    q[int(drafts[b, acc])] = 1.0
            else:
                q = dist(draft[b, acc])
            r = (p - q).clamp(min=0)
            if float(r.sum()) == 0:
                r = p
        run = r.cumsum(0)
        if float(run[-1]) == 0:
            pick = -1
        else:
            over = ((run > float(u[b, -1]) * run[-1]) & (r > 0)).nonzero()
            pick = int(over[0]) if len(over) else int((r > 0).nonzero()[-1])
        row = [int(v) for v in drafts[b, :acc]] + [pick]
        toks.append(row + [-1] * (n1 - len(row)))
        accs.append(acc)
    return toks, accs
