"""Keys and values on their way into a paged cache, and attention over a cache that holds them in 4 bits.

Four operators, each in a plain form (elementary torch operations) and through the framework's entry points:

* ``rotate``: the norms of each query's and key's head, the rotation by position, and the rows of a bf16 cache, from a
  fused projection's output;
* ``store``: key and value rows into a cache of 4 bits, and their values read back;
* ``decode``: attention of one new token a request over its pages of such a cache;
* ``chunk``: the same for each request's new tokens, causal over prefix and chunk.

4 bits: blocks of 32 dims, each value one of 0, 1/2, 1, 3/2, 2, 3, 4, 6 with a sign, times a power of two of its block's,
two values a byte (the even dim in the low bits) and a byte of exponent plus 127 a block.

Lengths come from a case's own ``lens_seed``, so a case's work does not depend on the seed of its values. Values are
N(0, 1) in bf16 before they are rounded to 4 bits; pages are scattered over the pool at random.
"""

from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False
DEV = torch.device("cuda:0")
EPS = 1e-6
POSITIONS = 40960  # of the rotation's table
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # a decode step's new tokens, one a request
        dict(name="rotate-decode", kind="rotate", tokens=64, q_heads=64, kv_heads=8, dim=128, rotary=128, interleaved=False, normed=True, page=64),
        # ragged chunks of a smaller model that rotates half of a head's dims, in pairs
        dict(name="rotate-chunk", kind="rotate", tokens=777, q_heads=28, kv_heads=4, dim=128, rotary=64, interleaved=True, normed=True, page=16),
        # the benchmark's chunked prefill: four chunks of 2048 tokens
        dict(name="rotate-prefill", kind="rotate", tokens=8192, q_heads=64, kv_heads=8, dim=128, rotary=128, interleaved=False, normed=True, page=64),
        # the rows of a decode step
        dict(name="store-decode", kind="store", tokens=64, kv_heads=8, dim=128, page=64),
        # the rows of four chunks of 2048 tokens
        dict(name="store-prefill", kind="store", tokens=8192, kv_heads=8, dim=128, page=64),
        # one user's chat, some 1,500 tokens in: the smallest decode call
        dict(name="decode-single", kind="decode", batch=1, q_heads=32, kv_heads=8, dim=128, page=16, lo=1400, hi=1600, lens_seed=7),
        # short contexts on a small model's heads, at the engine's default page size
        dict(name="decode-page1", kind="decode", batch=19, q_heads=14, kv_heads=2, dim=64, page=1, lo=100, hi=4000, lens_seed=2),
        # the benchmark's decode batch: 64 requests of 1k to 8k tokens
        dict(name="decode-batch", kind="decode", batch=64, q_heads=64, kv_heads=8, dim=128, page=64, lo=1024, hi=8192, lens_seed=0),
        # long documents on one of eight tensor-parallel ranks: one KV head
        dict(name="decode-long", kind="decode", batch=8, q_heads=8, kv_heads=1, dim=128, page=64, lo=32768, hi=131072, lens_seed=0),
        # short continuations of short chats, seven query heads to a KV head
        dict(name="chunk-short", kind="chunk", batch=3, q_heads=28, kv_heads=4, dim=128, page=16, elo=5, ehi=60, plo=0, phi=500, lens_seed=4),
        # drafted tokens checked against long contexts
        dict(name="chunk-draft", kind="chunk", batch=16, q_heads=32, kv_heads=8, dim=128, page=64, elo=1, ehi=8, plo=1024, phi=16384, lens_seed=5),
        # the benchmark's chunked prefill on prefixes of up to 8192
        dict(name="chunk-prefill", kind="chunk", batch=4, q_heads=64, kv_heads=8, dim=128, page=64, elo=2048, ehi=2048, plo=0, phi=8192, lens_seed=6),
    ]


HEADS = [(8, 1), (8, 2), (28, 4), (16, 16), (32, 8), (40, 8), (64, 8), (12, 3), (14, 2)]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["rotate", "store", "decode", "decode", "chunk", "chunk"])
    while True:
        hq, hk = rng.choice(HEADS)
        heads = dict(q_heads=hq, kv_heads=hk, dim=rng.choice([64, 128]))
        page = 1 << rng.randrange(0, 8)
        if kind == "rotate":
            c = dict(kind=kind, tokens=_spread(rng, 1, 8192), **heads, rotary=rng.choice([heads["dim"], heads["dim"], heads["dim"] // 2]),
                     interleaved=rng.random() < 0.5, normed=rng.random() < 0.75, page=page)
            fits = c["tokens"] * (hq + hk) <= 8192 * 72
        elif kind == "store":
            c = dict(kind=kind, tokens=_spread(rng, 1, 8192), kv_heads=hk, dim=heads["dim"], page=page)
            fits = c["tokens"] * hk <= 8192 * 8
        elif kind == "decode":
            hi = _spread(rng, 2, 131072)
            c = dict(kind=kind, batch=_spread(rng, 1, 128), **heads, page=page, lo=max(1, hi // rng.choice([1, 8, 100])), hi=hi, lens_seed=rng.randrange(1 << 30))
            fits = c["batch"] * hk * hi <= 64 * 8 * 8192
        else:
            ehi, phi = _spread(rng, 2, 4096), _spread(rng, 1, 32768)
            c = dict(kind=kind, batch=_spread(rng, 1, 32), **heads, page=page, elo=max(1, ehi // rng.choice([1, 4, 50])), ehi=ehi,
                     plo=phi // rng.choice([1, 4, 50]), phi=phi, lens_seed=rng.randrange(1 << 30))
            fits = c["batch"] * hq * ehi * (ehi + phi) <= 4 * 64 * 2048 * 10240 and c["batch"] * hk * (ehi + phi) <= 64 * 8 * 8192
        if fits:
            return c


def lengths(case):
    """(new tokens, keys) of each request."""
    r = random.Random(case["lens_seed"])
    n = case["batch"]
    if case["kind"] == "decode":
        return [1] * n, [r.randint(case["lo"], case["hi"]) for _ in range(n)]
    e = [r.randint(case["elo"], case["ehi"]) for _ in range(n)]
    return e, [x + r.randint(case["plo"], case["phi"]) for x in e]


def work(case):
    d, hk = case["dim"], case["kv_heads"]
    packed = d // 2 + d // 32  # bytes of a row of 4 bits
    if case["kind"] == "rotate":
        t, hq = case["tokens"], case["q_heads"]
        # the projection's rows read and written, positions, slots, and a row of the table each
        return {"bytes": t * ((hq + 2 * hk) * d * 4 + 8 + 4 * case["rotary"]), "flops": t * (hq + hk) * (4 * d + 3 * case["rotary"])}
    if case["kind"] == "store":
        # rows read, their 4 bits written, their values written; slots
        return {"bytes": case["tokens"] * (2 * hk * (2 * d + packed + 2 * d) + 4), "flops": 0}
    e, l = lengths(case)
    hq, new, keys = case["q_heads"], sum(e), sum(l)
    pairs = sum(y * (x - y) + y * (y + 1) // 2 for x, y in zip(l, e))
    table = 4 * sum(-(-x // case["page"]) for x in l)
    return {"bytes": 4 * new * hq * d + 4 * new * hq + 2 * keys * hk * packed + table + 4 * case["batch"], "flops": 4 * d * hq * pairs}


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _cumulative(x):
    out = [0]
    for v in x:
        out.append(out[-1] + v)
    return out


def _to_4_bits(x):
    """Codes ``[..., D / 2]`` and exponents ``[..., D / 32]`` of rows ``x [..., D]``: a block's exponent is its largest
    magnitude's, less 2, so that this lies in [4, 8) units; values are rounded to the nearest, ties to even, 6 at most."""
    b = x.float().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1)
    e = (torch.frexp(top).exponent - 3).clamp_min(-127)
    e = torch.where(top == 0, -127, e)
    y = torch.ldexp(b, -e[..., None])
    m = y.abs()
    code = sum((m > t).to(torch.uint8) for t in (0.25, 1.25, 2.5, 5.0)) + sum((m >= t).to(torch.uint8) for t in (0.75, 1.75, 3.5))
    code = (code + 8 * (y < 0).to(torch.uint8)).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), (e + 127).to(torch.uint8)


def _values(codes, scales):
    """The values of rows in 4 bits, in 32."""
    table = torch.tensor(MAGNITUDES + tuple(-x for x in MAGNITUDES), device=DEV)
    v = torch.stack((table[(codes & 15).long()], table[(codes >> 4).long()]), -1).flatten(-2)
    return torch.ldexp(v.unflatten(-1, (-1, 32)), (scales.int() - 127)[..., None]).flatten(-2)


def _cos_sin(rotary):
    inv = 50000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device=DEV) / rotary)
    angle = torch.arange(POSITIONS, dtype=torch.float64, device=DEV)[:, None] * inv
    return torch.cat((angle.cos(), angle.sin()), 1).float()


def _pool4(pages, ps, hk, d):
    """An empty pool of 4 bits ``[pages, ps, Hkv, ...]``, a head's rows of a page next to each other."""
    return [torch.zeros((pages, hk, ps, w), dtype=torch.uint8, device=DEV).transpose(1, 2) for w in (d // 2, d // 32)]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    kind, hk, d, ps = case["kind"], case["kv_heads"], case["dim"], case["page"]

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEV, dtype=torch.bfloat16)

    s = {"kind": kind, "page": ps}
    if kind in ("rotate", "store"):
        t = case["tokens"]
        pages = -(-t // ps) + 3
        s["slots"] = torch.randperm(pages * ps, generator=g, device=DEV)[:t].to(torch.int32)
        if kind == "store":
            s.update(k=normal(t, hk, d), v=normal(t, hk, d), k_pool=_pool4(pages, ps, hk, d), v_pool=_pool4(pages, ps, hk, d))
            return s
        hq = case["q_heads"]
        qkv = normal(t, hq + 2 * hk, d)
        s.update(q=qkv[:, :hq], k=qkv[:, hq : hq + hk], v=qkv[:, hq + hk :], interleaved=case["interleaved"],
                 positions=torch.randint(0, POSITIONS, (t,), generator=g, device=DEV).to(torch.int32), cos_sin=_cos_sin(case["rotary"]),
                 q_weight=1 + 0.1 * normal(d) if case["normed"] else None, k_weight=1 + 0.1 * normal(d) if case["normed"] else None,
                 q_out=torch.zeros((t, hq, d), dtype=torch.bfloat16, device=DEV), k_pool=torch.zeros((pages, ps, hk, d), dtype=torch.bfloat16, device=DEV),
                 v_pool=torch.zeros((pages, ps, hk, d), dtype=torch.bfloat16, device=DEV))
        return s
    e, l = lengths(case)
    n, hq = case["batch"], case["q_heads"]
    need = [-(-x // ps) for x in l]
    pages = sum(need) + 8
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    first = torch.tensor(_cumulative(need)[:-1], device=DEV)[:, None] + torch.arange(max(need), device=DEV)
    s.update(batch=n, total=sum(e), max_e=max(e), max_l=max(l), keys=sum(l), scale=d ** -0.5, q=normal(sum(e), hq, d), cu=_i32(_cumulative(e)), lens=_i32(l),
             pt=order[first.clamp_max(pages - 1)].contiguous())
    for name in ("k_pool", "v_pool"):
        s[name] = _pool4(pages, ps, hk, d)
        part = max(1, (1 << 25) // (ps * hk * d))
        for p0 in range(0, pages, part):
            for whole, some in zip(s[name], _to_4_bits(normal(min(part, pages - p0), ps, hk, d))):
                whole[p0 : p0 + part] = some
    s.update(out=torch.empty_like(s["q"]), lse=torch.empty((sum(e), hq), dtype=torch.float32, device=DEV))
    return s


# ---- plain forms


def _plain_rotate(s):
    r = s["cos_sin"].shape[1]
    c, n = s["cos_sin"][s["positions"].long()].float()[:, None].chunk(2, -1)

    def turned(x, weight):
        x = x.float()
        if weight is not None:
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
        if s["interleaved"]:
            a, b = x[..., 0:r:2], x[..., 1:r:2]
            y = torch.stack((a * c - b * n, b * c + a * n), -1).flatten(-2)
        else:
            a, b = x[..., : r // 2], x[..., r // 2 : r]
            y = torch.cat((a * c - b * n, b * c + a * n), -1)
        return torch.cat((y, x[..., r:]), -1).bfloat16()

    slots = s["slots"].long()
    s["q_out"].copy_(turned(s["q"], s["q_weight"]))
    s["k_pool"].flatten(0, 1)[slots] = turned(s["k"], s["k_weight"])
    s["v_pool"].flatten(0, 1)[slots] = s["v"]
    return {"q": s["q_out"], "k_pool": s["k_pool"], "v_pool": s["v_pool"]}


def _plain_store(s):
    page, at = s["slots"].long() // s["page"], s["slots"].long() % s["page"]
    out = {}
    for name in ("k", "v"):
        codes, scales = s[name + "_pool"]
        codes[page, at], scales[page, at] = _to_4_bits(s[name])
        out[name] = _values(codes[page, at], scales[page, at]).bfloat16()
    return out


def _plain_attend(s):
    """``q [T, Hq, D]`` over the requests' keys, padded to the longest, causal at the end of each request's."""
    j = torch.arange(s["max_l"], device=DEV)
    page, at = s["pt"][:, j // s["page"]].long(), j % s["page"]
    k, v = (_values(codes[page, at], scales[page, at]) for codes, scales in (s["k_pool"], s["v_pool"]))
    n, e, l, q, cu, lens = s["batch"], s["max_e"], s["max_l"], s["q"], s["cu"], s["lens"]
    hq, d = q.shape[1:]
    hk = k.shape[2]
    ext = cu[1:] - cu[:-1]
    i = torch.arange(e, device=DEV)
    rows = (cu[:-1, None] + i).clamp_max(q.shape[0] - 1).long()
    qp = q[rows].float().view(n, e, hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(n, hk, -1, d)
    x = torch.matmul(qp, k.permute(0, 2, 3, 1)).view(n, hk, hq // hk, e, l).mul_(s["scale"])
    past = j > ((lens - ext)[:, None] + i)[:, :, None]
    x.masked_fill_(past[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x.sub_(top).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(n, hk, -1, l), v.permute(0, 2, 1, 3)).view(n, hk, hq // hk, e, d) / total
    lse = (top + total.log()).squeeze(-1)
    b = torch.repeat_interleave(torch.arange(n, device=DEV), ext, output_size=s["total"])
    t = torch.arange(s["total"], device=DEV) - cu[b]
    return o.permute(0, 3, 1, 2, 4)[b, t].reshape(-1, hq, d).to(q.dtype), lse.permute(0, 3, 1, 2)[b, t].reshape(-1, hq)


# ---- the framework's calls


def _lib():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mini-sglang_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from minisgl_amd.kernel import lib

    return lib


def _own(s):
    lib = _lib()
    if s["kind"] == "rotate":
        lib.qk_norm_rope(s["q"], s["k"], s["v"], s["q_weight"], s["k_weight"], EPS, s["positions"], s["cos_sin"], s["interleaved"], s["q_out"],
                         s["k_pool"], s["v_pool"], slots=s["slots"])
        return {"q": s["q_out"], "k_pool": s["k_pool"], "v_pool": s["v_pool"]}
    k_pool, v_pool = lib.MX4Pool(*s["k_pool"]), lib.MX4Pool(*s["v_pool"])
    if s["kind"] == "store":
        lib.mx4_store(k_pool, v_pool, s["slots"], s["k"], s["v"])
        k, v = lib.mx4_load(k_pool, v_pool, s["slots"])
        return {"k": k, "v": v}
    if s["kind"] == "decode":
        lib.gqa_decode_mx4(s["q"], k_pool, v_pool, s["pt"], s["lens"], s["scale"], s["out"], s["lse"])
    else:
        lib.gqa_chunk_mx4(s["q"], k_pool, v_pool, s["pt"], s["cu"], s["lens"], s["max_e"], s["scale"], s["out"], s["lse"], total_keys=s["keys"])
    return s["out"], s["lse"]


def run(s):
    if own:
        return _own(s)
    if s["kind"] == "rotate":
        return _plain_rotate(s)
    return _plain_store(s) if s["kind"] == "store" else _plain_attend(s)


# ---- in 64 bits


def _exact_values(codes, scales):
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
    # sign, two bits of exponent and one of mantissa
    e, m = (c >> 1) & 3, (c & 1).double()
    size = torch.where(e == 0, 0.5 * m, (1 + 0.5 * m) * 2.0 ** (e - 1).double())
    unit = 2.0 ** (scales.double() - 127)
    return torch.where(c >= 8, -size, size) * unit.repeat_interleave(32, -1)


def _exact_rounded(x):
    """Rows ``x [T, H, D]`` as 4 bits hold them, value by value: the nearest of the block's, of two alike the one with an even code."""
    b = x.double().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True)
    unit = torch.where(top > 0, 2.0 ** torch.floor(torch.log2(top)), 1.0) / 4
    grid = torch.tensor(MAGNITUDES, dtype=torch.float64, device=DEV)
    best, off = torch.zeros_like(b), torch.full_like(b, math.inf)
    for c in (0, 2, 4, 6, 1, 3, 5, 7):
        far = (b.abs() - grid[c] * unit).abs()
        best, off = torch.where(far < off, grid[c] * unit, best), torch.minimum(far, off)
    return (torch.sign(b) * best).flatten(-2)


def _exact_rotate(s):
    r = s["cos_sin"].shape[1]
    at = s["cos_sin"].double()[s["positions"].long()]
    turn = torch.complex(at[:, : r // 2], at[:, r // 2 :])[:, None]

    def turned(x, weight):
        x = x.double()
        if weight is not None:
            x = weight.double() * x * torch.rsqrt(x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS)
        first, second = (slice(0, r, 2), slice(1, r, 2)) if s["interleaved"] else (slice(0, r // 2), slice(r // 2, r))
        z = torch.complex(x[..., first], x[..., second]) * turn
        x[..., first], x[..., second] = z.real, z.imag
        return x

    pools = []
    for rows, pool in ((turned(s["k"].clone(), s["k_weight"]), s["k_pool"]), (s["v"].double(), s["v_pool"])):
        flat = torch.zeros(pool.shape, dtype=torch.float64, device=DEV).view(-1, *pool.shape[2:])
        flat[s["slots"].long()] = rows
        pools.append(flat.view(pool.shape))
    return {"q": turned(s["q"].clone(), s["q_weight"]), "k_pool": pools[0], "v_pool": pools[1]}


def exact(case, seed):
    """Attention: each request and KV head by itself."""
    s = prepare(case, seed)
    if s["kind"] == "rotate":
        return _exact_rotate(s)
    if s["kind"] == "store":
        return {"k": _exact_rounded(s["k"]), "v": _exact_rounded(s["v"])}
    e, l = lengths(case)
    hq, hk, d, ps = case["q_heads"], case["kv_heads"], case["dim"], case["page"]
    group, q = hq // hk, s["q"]
    out = torch.empty((s["total"], hq, d), dtype=torch.float64, device=DEV)
    lse = torch.empty((s["total"], hq), dtype=torch.float64, device=DEV)
    t0 = 0
    for b in range(case["batch"]):
        rows = slice(t0, t0 + e[b])
        pages = s["pt"][b, : -(-l[b] // ps)].long()
        hidden = torch.ones((e[b], l[b]), dtype=torch.bool, device=DEV).triu(l[b] - e[b] + 1)
        for h in range(hk):
            heads = slice(h * group, (h + 1) * group)
            k, v = (_exact_values(codes[pages, :, h], scales[pages, :, h]).flatten(0, 1)[: l[b]] for codes, scales in (s["k_pool"], s["v_pool"]))
            x = torch.einsum("ihd,jd->hij", q[rows, heads].double(), k) * (1.0 / math.sqrt(d))
            x = x.masked_fill(hidden, -math.inf)
            z = torch.logsumexp(x, -1, keepdim=True)
            out[rows, heads] = torch.matmul(torch.exp(x - z), v).transpose(0, 1)
            lse[rows, heads] = z.squeeze(-1).transpose(0, 1)
        t0 += e[b]
    return out, lse
