"""64-bit oracle of the grouped-head attention and of a step's tables. TEST INFRASTRUCTURE ONLY.

Attention: query i (of E) of a request with L keys attends keys ``j <= L - E + i``, query head h reads KV head
``h // (Hq / Hkv)``; ``s_j = scale <q, k_j>``, ``lse = ln sum_j exp(s_j)``, ``o = sum_j exp(s_j - lse) v_j``; a query
without keys gives ``o = 0``, ``lse = -inf`` (semantics of the reference's call, python/minisgl/attention/fa.py:84-97,
155-182).

Tables: a step's page allocation, slots and positions (python/minisgl/scheduler/cache.py:42-53,119-161 and
scheduler/scheduler.py:198-214) and its page table (attention/fa.py:92-97), request by request.
"""

from __future__ import annotations

from typing import List, NamedTuple

import torch


class Attention(NamedTuple):
    out: torch.Tensor  # float64 [E, Hq, D]
    lse: torch.Tensor  # float64 [E, Hq]
    out_bound: torch.Tensor  # how far a bf16 result may be from ``out``
    lse_bound: torch.Tensor  # how far an fp32 result may be from ``lse``


def attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float) -> Attention:
    """One request: ``q [E, Hq, D]``, ``k``, ``v [L, Hkv, D]``.

    The bounds, for a kernel that multiplies bf16 operands with fp32 sums, rounds the softmax numerators to bf16
    (half a step: 2^-8 of each) and the result to bf16:

    * a score's error is at most (D + 16) 2^-24 S, S = scale * max_j sum_d |q_d k_jd| (D roundings of a sum and a few
      of the scaling), and moves each numerator by as much, relatively: delta;
    * with A = sum_j softmax_j |v_j|: out is off by 2^-8 A (numerators), 2 delta A (scores, above and below the
      fraction), 2 (L + 16) 2^-24 A (sums over keys), and 2^-8 |out| (the last rounding); 2 % for second-order terms;
    * lse is off by delta + (L + 16) 2^-24 (the sum's logarithm) + 2^-22 |lse| (its own roundings).
    """
    E, Hq, D = q.shape
    L, Hkv, _ = k.shape
    out = torch.zeros((E, Hq, D), dtype=torch.float64)
    lse = torch.full((E, Hq), -float("inf"), dtype=torch.float64)
    ob, lb = torch.zeros_like(out), torch.zeros_like(lse)
    if E == 0 or L == 0:
        return Attention(out, lse, ob, lb)
    seen = torch.arange(L) <= (L - E + torch.arange(E))[:, None]
    for h in range(Hq):
        kh, vh, qh = k[:, h // (Hq // Hkv)].double(), v[:, h // (Hq // Hkv)].double(), q[:, h].double()
        s = torch.where(seen, qh @ kh.t() * scale, -float("inf"))
        z = torch.logsumexp(s, -1)
        some = seen.any(-1)
        p = torch.where(seen & some[:, None], torch.exp(s - torch.where(some, z, 0.0)[:, None]), 0.0)
        vv = torch.where(seen.any(0)[:, None], vh, 0.0)
        out[:, h], lse[:, h] = p @ vv, z
        size = torch.where(seen, (qh.abs() @ kh.abs().t()) * scale, 0.0).amax(-1)
        delta = (D + 16) * 2.0 ** -24 * size
        a = p @ vv.abs()
        ob[:, h] = 1.02 * ((2.0 ** -8 + 2 * delta + 2 * (L + 16) * 2.0 ** -24)[:, None] * a + 2.0 ** -8 * out[:, h].abs())
        lb[:, h] = torch.where(some, delta + (L + 16) * 2.0 ** -24 + 2.0 ** -22 * z.abs(), 0.0)
    return Attention(out, lse, ob, lb)


def prompt(q, k, v, lens: List[int], scale: float) -> Attention:
    """Packed prompts of ``lens`` tokens."""
    parts, t = [], 0
    for n in lens:
        parts.append(attend(q[t : t + n], k[t : t + n], v[t : t + n], scale))
        t += n
    return Attention(*(torch.cat(x) for x in zip(*parts)))


def chunk(q, k_pool, v_pool, page_table, extends: List[int], lens: List[int], scale: float) -> Attention:
    """The last ``extends[b]`` tokens of each request over its ``lens[b]`` keys in pages."""
    ps = k_pool.shape[1]
    kf, vf = k_pool.reshape(-1, *k_pool.shape[2:]), v_pool.reshape(-1, *v_pool.shape[2:])
    parts, t = [], 0
    for b, (e, n) in enumerate(zip(extends, lens)):
        j = torch.arange(n)
        rows = page_table[b].long()[j // ps] * ps + j % ps
        parts.append(attend(q[t : t + e], kf[rows], vf[rows], scale))
        t += e
    return Attention(*(torch.cat(x) for x in zip(*parts)))


class Tables(NamedTuple):
    token_table: torch.Tensor
    page_table: torch.Tensor
    out_loc: List[int]
    positions: List[int]
    cu_seqlens_q: List[int]
    pages_taken: int


def step_tables(token_table, table_idx, cached, device, free_slots, page_size: int, cols: int, alloc: int) -> Tables:
    table = token_table.clone()
    pages = torch.zeros((len(cached), cols), dtype=torch.int32)
    loc, pos, cu, taken = [], [], [0], 0
    for b, (row, c, d) in enumerate(zip(table_idx, cached, device)):
        if b < alloc:
            for j in range(-(-c // page_size), -(-d // page_size)):
                slot = int(free_slots[taken])
                taken += 1
                for i in range(min(page_size, table.shape[1] - j * page_size)):
                    table[row, j * page_size + i] = slot + i
        for j in range(-(-d // page_size)):
            pages[b, j] = int(table[row, j * page_size]) // page_size
        loc += [int(x) for x in table[row, c:d]]
        pos += list(range(c, d))
        cu.append(cu[-1] + d - c)
    return Tables(table, pages, loc, pos, cu, taken)
