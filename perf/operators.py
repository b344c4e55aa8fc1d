"""Attention with grouped heads over packed prompts and over a paged K/V cache, and the tables that address the cache.

Four operators, each in a plain form (elementary torch operations) and through the framework's entry points:

* ``prompt``: causal attention over whole prompts, packed sequences of different lengths;
* ``chunk``: attention of each request's new tokens over its pages of a K/V cache, causal over prefix and chunk;
* ``decode``: the same for one new token a request;
* ``tables``: page tables, token table rows, slots and positions of a step, from the requests' lengths.

Lengths come from a case's own ``lens_seed``, so a case's work does not depend on the seed of its values.
Values are N(0, 1) in bf16; pages are scattered over the pool at random.
"""

from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False
DEV = torch.device("cuda:0")


def listed():
    return [
        # a handful of short prompts on a small model's heads: latency and launches
        dict(name="prompt-short", kind="prompt", batch=7, q_heads=8, kv_heads=2, dim=64, lo=1, hi=300, lens_seed=1),
        # ordinary prompts of different lengths, arriving together
        dict(name="prompt-ragged", kind="prompt", batch=6, q_heads=32, kv_heads=8, dim=128, lo=200, hi=2000, lens_seed=2),
        # two long documents
        dict(name="prompt-long", kind="prompt", batch=2, q_heads=64, kv_heads=8, dim=128, lo=7700, hi=8192, lens_seed=3),
        # short continuations of short chats, seven query heads to a KV head, small pages
        dict(name="chunk-short", kind="chunk", batch=3, q_heads=28, kv_heads=4, dim=128, page=16, elo=5, ehi=60, plo=0,
             phi=500, lens_seed=4),
        # drafted tokens checked against long contexts, at the engine's default page size
        dict(name="chunk-draft", kind="chunk", batch=16, q_heads=32, kv_heads=8, dim=128, page=1, elo=1, ehi=8, plo=1024,
             phi=16384, lens_seed=5),
        # the benchmark's chunked prefill: four chunks of 2048 tokens on prefixes of up to 8192
        dict(name="chunk-prefill", kind="chunk", batch=4, q_heads=64, kv_heads=8, dim=128, page=64, elo=2048, ehi=2048,
             plo=0, phi=8192, lens_seed=6),
        # one user's chat, some 1,500 tokens in: the smallest decode call
        dict(name="decode-single", kind="decode", batch=1, q_heads=32, kv_heads=8, dim=128, page=16, lo=1400, hi=1600,
             lens_seed=7),
        # the benchmark's decode batch: 64 requests of 1k to 8k tokens
        dict(name="decode-batch", kind="decode", batch=64, q_heads=64, kv_heads=8, dim=128, page=64, lo=1024, hi=8192,
             lens_seed=0),
        # long documents on one of eight tensor-parallel ranks: one KV head
        dict(name="decode-long", kind="decode", batch=8, q_heads=8, kv_heads=1, dim=128, page=64, lo=32768, hi=131072,
             lens_seed=0),
        # the tables of a decode step
        dict(name="tables-decode", kind="tables", batch=64, page=16, elo=1, ehi=1, plo=1024, phi=8191, cols=8192,
             lens_seed=8),
        # the tables of a step of chunks on cached prefixes
        dict(name="tables-chunks", kind="tables", batch=61, page=64, elo=1, ehi=2048, plo=0, phi=8192, cols=16384,
             lens_seed=9),
        # many new prompts at once, at the engine's default page size
        dict(name="tables-prompts", kind="tables", batch=256, page=1, elo=1, ehi=8192, plo=0, phi=0, cols=8192,
             lens_seed=10),
    ]


HEADS = [(8, 1), (8, 2), (28, 4), (16, 16), (32, 8), (40, 8), (64, 8), (12, 3)]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["prompt", "chunk", "decode", "tables"])
    while True:
        seed = rng.randrange(1 << 30)
        hq, hk = rng.choice(HEADS)
        heads = dict(q_heads=hq, kv_heads=hk, dim=rng.choice([64, 128]))
        if kind == "prompt":
            hi = _spread(rng, 20, 8192)
            c = dict(kind=kind, batch=_spread(rng, 1, 32), **heads, lo=max(1, hi // rng.choice([1, 3, 20])), hi=hi, lens_seed=seed)
            # padded scores of the plain form
            fits = c["batch"] * hq * hi * hi <= 2 * 64 * 8192 * 8192
        elif kind == "chunk":
            ehi, phi = _spread(rng, 2, 4096), _spread(rng, 1, 32768)
            c = dict(kind=kind, batch=_spread(rng, 1, 32), **heads, page=1 << rng.randrange(0, 8), elo=max(1, ehi // rng.choice([1, 4, 50])),
                     ehi=ehi, plo=phi // rng.choice([1, 4, 50]), phi=phi, lens_seed=seed)
            fits = (c["batch"] * hq * ehi * (ehi + phi) <= 4 * 64 * 2048 * 10240
                    and c["batch"] * hk * (ehi + phi) <= 64 * 8 * 8192)
        elif kind == "decode":
            hi = _spread(rng, 2, 131072)
            c = dict(kind=kind, batch=_spread(rng, 1, 128), **heads, page=1 << rng.randrange(0, 8), lo=max(1, hi // rng.choice([1, 8, 100])), hi=hi,
                     lens_seed=seed)
            fits = c["batch"] * hk * hi <= 64 * 8 * 8192
        else:
            ehi, phi = _spread(rng, 1, 8192), _spread(rng, 1, 8192)
            c = dict(kind=kind, batch=_spread(rng, 1, 256), page=1 << rng.randrange(0, 8), elo=max(1, ehi // rng.choice([1, 4, 50])), ehi=ehi,
                     plo=phi // rng.choice([1, 4, 50]), phi=phi, cols=-(-(ehi + phi) // 256) * 256, lens_seed=seed)
            fits = c["batch"] * ehi <= 256 * 8192
        if fits:
            return c


def lengths(case):
    """(new tokens, keys) of each request."""
    r = random.Random(case["lens_seed"])
    n, kind = case["batch"], case["kind"]
    if kind == "prompt":
        e = [r.randint(case["lo"], case["hi"]) for _ in range(n)]
        return e, list(e)
    if kind == "decode":
        return [1] * n, [r.randint(case["lo"], case["hi"]) for _ in range(n)]
    e = [r.randint(case["elo"], case["ehi"]) for _ in range(n)]
    return e, [x + r.randint(case["plo"], case["phi"]) for x in e]


def work(case):
    e, l = lengths(case)
    new, keys = sum(e), sum(l)
    if case["kind"] == "tables":
        ps = case["page"]
        pages = sum(-(-x // ps) for x in l)
        fresh = sum(-(-x // ps) - -(-(x - y) // ps) for x, y in zip(l, e))
        # lengths, rows, free slots and the old pages' entries read; token table rows, the page table, slots,
        # positions and offsets written
        table = case["batch"] * -(-max(l) // ps)
        return {"bytes": 4 * (3 * case["batch"] + pages + fresh * ps + table + 2 * new + case["batch"]), "flops": 0}
    hq, hk, d = case["q_heads"], case["kv_heads"], case["dim"]
    pairs = sum(y * (x - y) + y * (y + 1) // 2 for x, y in zip(l, e))
    table = 0 if case["kind"] == "prompt" else 4 * sum(-(-x // case["page"]) for x in l)
    return {"bytes": 4 * new * hq * d + 4 * new * hq + 4 * keys * hk * d + table + 4 * case["batch"], "flops": 4 * d * hq * pairs}


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _cumulative(x):
    out = [0]
    for v in x:
        out.append(out[-1] + v)
    return out


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    e, l = lengths(case)
    n, kind = case["batch"], case["kind"]
    s = {"kind": kind, "batch": n, "total": sum(e), "max_e": max(e), "max_l": max(l)}
    if kind == "tables":
        ps, cols = case["page"], case["cols"]
        held = [-(-(x - y) // ps) for x, y in zip(l, e)]  # pages that the cached tokens lie in
        fresh = sum(-(-x // ps) for x in l) - sum(held)
        order = torch.randperm(sum(held) + fresh + 64, generator=g, device=DEV).to(torch.int32) * ps
        table = torch.zeros((n + 5, -(-cols // ps) * ps), dtype=torch.int32, device=DEV)
        rows = torch.randperm(n + 5, generator=g, device=DEV)[:n]
        at = _cumulative(held)
        span = torch.arange(max(max(held), 1), device=DEV)
        first = torch.tensor(at[:-1], device=DEV)[:, None] + span
        inside = span < torch.tensor(held, device=DEV)[:, None]
        slots = torch.where(inside, order[first.clamp_max(order.numel() - 1)], torch.zeros((), dtype=torch.int32, device=DEV))
        tokens = (slots[:, :, None] + torch.arange(ps, dtype=torch.int32, device=DEV)) * inside[:, :, None]
        table[rows, : span.numel() * ps] = tokens.flatten(1).to(torch.int32)
        s.update(page=ps, token_table=table, table_idx=rows.to(torch.int32), cached=_i32([x - y for x, y in zip(l, e)]), device=_i32(l),
                 free=order[sum(held):].contiguous(), cols=-(-max(l) // ps))
        return s
    hq, hk, d = case["q_heads"], case["kv_heads"], case["dim"]

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEV, dtype=torch.bfloat16)

    s.update(scale=d ** -0.5, q=normal(sum(e), hq, d), cu=_i32(_cumulative(e)), lens=_i32(l))
    if kind == "prompt":
        s.update(k=normal(sum(e), hk, d), v=normal(sum(e), hk, d))
    else:
        ps = case["page"]
        need = [-(-x // ps) for x in l]
        pages = sum(need) + 8
        order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
        first = torch.tensor(_cumulative(need)[:-1], device=DEV)[:, None] + torch.arange(max(need), device=DEV)
        s.update(page=ps, k=normal(pages, ps, hk, d), v=normal(pages, ps, hk, d), pt=order[first.clamp_max(pages - 1)].contiguous())
    s.update(out=torch.empty_like(s["q"]), lse=torch.empty((sum(e), hq), dtype=torch.float32, device=DEV))
    return s


# ---- plain forms


def _attend(q, k, v, cu, lens, s):
    """``q [T, Hq, D]`` over padded ``k, v [B, L, Hkv, D]``, causal at the end of each request's keys."""
    n, e, l = s["batch"], s["max_e"], s["max_l"]
    hq, d = q.shape[1:]
    hk = k.shape[2]
    ext = cu[1:] - cu[:-1]
    i, j = torch.arange(e, device=DEV), torch.arange(l, device=DEV)
    rows = (cu[:-1, None] + i).clamp_max(q.shape[0] - 1).long()
    qp = q[rows].float().view(n, e, hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(n, hk, -1, d)
    kp = k.permute(0, 2, 3, 1).float()
    x = torch.matmul(qp, kp).view(n, hk, hq // hk, e, l).mul_(s["scale"])
    past = j > ((lens - ext)[:, None] + i)[:, :, None]
    x.masked_fill_(past[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x.sub_(top).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(n, hk, -1, l), v.permute(0, 2, 1, 3).float()).view(n, hk, hq // hk, e, d) / total
    lse = (top + total.log()).squeeze(-1)
    b = torch.repeat_interleave(torch.arange(n, device=DEV), ext, output_size=s["total"])
    t = torch.arange(s["total"], device=DEV) - cu[b]
    return o.permute(0, 3, 1, 2, 4)[b, t].reshape(-1, hq, d).to(q.dtype), lse.permute(0, 3, 1, 2)[b, t].reshape(-1, hq)


def _plain_prompt(s):
    at = (s["cu"][:-1, None] + torch.arange(s["max_l"], device=DEV)).clamp_max(s["total"] - 1).long()
    return _attend(s["q"], s["k"][at], s["v"][at], s["cu"], s["lens"], s)


def _plain_paged(s):
    ps = s["page"]
    j = torch.arange(s["max_l"], device=DEV)
    at = (s["pt"][:, j // ps] * ps + j % ps).long()
    k, v = s["k"].flatten(0, 1), s["v"].flatten(0, 1)
    return _attend(s["q"], k[at], v[at], s["cu"], s["lens"], s)


def _plain_tables(s):
    ps, n, table, rows = s["page"], s["batch"], s["token_table"], s["table_idx"].long()
    c, d = s["cached"].long(), s["device"].long()
    first, last = (c + ps - 1) // ps, (d + ps - 1) // ps
    j = torch.arange(s["cols"], device=DEV)
    fresh = (j >= first[:, None]) & (j < last[:, None])
    base = torch.cumsum(last - first, 0) - (last - first)
    slot = s["free"][torch.where(fresh, base[:, None] + j - first[:, None], 0)]
    width = s["cols"] * ps
    tokens = (slot[:, :, None] + torch.arange(ps, dtype=torch.int32, device=DEV)).flatten(1)
    table[rows, :width] = torch.where(fresh.repeat_interleave(ps, 1), tokens, table[rows, :width])
    pages = torch.where(j < last[:, None], table[rows, : width : ps] // ps, 0).to(torch.int32)
    cu = torch.cat((torch.zeros(1, dtype=torch.int64, device=DEV), torch.cumsum(d - c, 0)))
    b = torch.repeat_interleave(torch.arange(n, device=DEV), d - c, output_size=s["total"])
    pos = c[b] + torch.arange(s["total"], device=DEV) - cu[b]
    return {"token_table": table, "page_table": pages, "out_loc": table[rows[b], pos], "positions": pos.to(torch.int32), "cu_seqlens_q": cu.to(torch.int32)}


# ---- the framework's calls


def _lib():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mini-sglang_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from minisgl_amd.kernel import lib

    return lib


def _own(s):
    lib, kind = _lib(), s["kind"]
    if kind == "tables":
        t = lib.page_tables_from_lengths(s["token_table"], s["table_idx"], s["cached"], s["device"], s["free"], s["page"], s["max_l"], s["max_e"], s["total"])
        return {"token_table": s["token_table"], "page_table": t.page_table, "out_loc": t.out_loc, "positions": t.positions, "cu_seqlens_q": t.cu_seqlens_q}
    out, lse = s["out"], s["lse"]
    if kind == "prompt":
        lib.gqa_prompt(s["q"], s["k"], s["v"], s["cu"], s["scale"], out, lse)
    elif kind == "chunk":
        lib.gqa_chunk(s["q"], s["k"], s["v"], s["pt"], s["cu"], s["lens"], s["max_e"], s["scale"], out, lse)
    else:
        lib.gqa_decode(s["q"], s["k"], s["v"], s["pt"], s["lens"], s["scale"], out, lse)
    return out, lse


def run(s):
    if own:
        return _own(s)
    if s["kind"] == "tables":
        return _plain_tables(s)
    return _plain_prompt(s) if s["kind"] == "prompt" else _plain_paged(s)


def exact(case, seed):
    """Each request and KV head by itself, in 64 bits."""
    s = prepare(case, seed)
    if s["kind"] == "tables":
        return None
    e, l = lengths(case)
    hq, hk, d = case["q_heads"], case["kv_heads"], case["dim"]
    group = hq // hk
    q, k, v = s["q"], s["k"].reshape(-1, hk, d), s["v"].reshape(-1, hk, d)
    out = torch.empty((s["total"], hq, d), dtype=torch.float64, device=DEV)
    lse = torch.empty((s["total"], hq), dtype=torch.float64, device=DEV)
    t0 = 0
    for b in range(case["batch"]):
        rows = slice(t0, t0 + e[b])
        if case["kind"] == "prompt":
            at = torch.arange(t0, t0 + l[b], device=DEV)
        else:
            ps = case["page"]
            at = (s["pt"][b, : -(-l[b] // ps), None].long() * ps + torch.arange(ps, device=DEV)).flatten()[: l[b]]
        hidden = torch.ones((e[b], l[b]), dtype=torch.bool, device=DEV).triu(l[b] - e[b] + 1)
        for h in range(hk):
            heads = slice(h * group, (h + 1) * group)
            x = torch.einsum("ihd,jd->hij", q[rows, heads].double(), k[at, h].double()) * (1.0 / math.sqrt(d))
            x = x.masked_fill(hidden, -math.inf)
            z = torch.logsumexp(x, -1, keepdim=True)
            out[rows, heads] = torch.matmul(torch.exp(x - z), v[at, h].double()).transpose(0, 1)
            lse[rows, heads] = z.squeeze(-1).transpose(0, 1)
        t0 += e[b]
    return out, lse
