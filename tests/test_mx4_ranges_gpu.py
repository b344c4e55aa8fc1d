"""Attention over the 4-bit cache at the ends of the numbers' range: scores far past 2^24, whose fp32 spacing is more than one,
and values whose sums come near fp32's largest. Bounds: as the bf16 cache's (test_gqa_ranges_gpu.py), of the codes' values."""

from __future__ import annotations

import pytest
import torch

from oracle import ref_mx4 as M
from test_gqa_ranges_gpu import Exact, far, huge, rising_scores
from test_mx4_gpu import Paged

pytestmark = pytest.mark.gpu

# streamed in 16 and 32 rows, split and joined, and in one piece; laid out
BATCHES = [([1, 1], [3000, 40], (8, 2)), ([3, 2], [5000, 600], (16, 4)), ([9], [300], (8, 2)), ([200, 3], [1500, 700], (8, 2)), ([300, 40], [300, 64], (6, 2))]


def fill(c, b, at, q, k, v):
    """Request b's queries, keys and values; (rows of the batch, queries, the values that the cache holds)."""
    e, n = c.extends[b], c.lens[b]
    c.q[at : at + e] = q
    c.put(c.k, b, range(n), k)
    c.put(c.v, b, range(n), v)
    return slice(at, at + e), q, M.values(*M.rounded(k)), M.values(*M.rounded(v))


@pytest.mark.parametrize("extends,prefixes,heads", BATCHES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page_size", [16, 64])
def test_far_scores(extends, prefixes, heads, dim, page_size):
    """One key of the prefix wins for either sign."""
    gen = torch.Generator().manual_seed(dim + len(extends))
    c = Paged(extends, prefixes, *heads, dim, page_size, seed=dim, scale=0.125)
    made, at = [], 0
    for b, (e, n) in enumerate(zip(extends, c.lens)):
        q, k = far(gen, e, heads[0], n, heads[1], dim)
        one = k.abs().amax((0, 1)).argmax()
        k[..., one] *= 0.25
        k[prefixes[b] // 3, :, one], k[prefixes[b] // 2, :, one] = 24576.0, -24576.0
        made.append(fill(c, b, at, q, k, torch.randn((n, heads[1], dim), generator=gen).to(torch.bfloat16)))
        at += e
    out, lse = c.run()
    for one, q, k, v in made:
        Exact(q, k, v, 0.125).check(out[one], lse[one])


@pytest.mark.parametrize("extends,prefixes,heads", BATCHES)
@pytest.mark.parametrize("dim", [64, 128])
def test_keys_alike_at_far_scores_weigh_alike(extends, prefixes, heads, dim):
    gen = torch.Generator().manual_seed(dim)
    c = Paged(extends, prefixes, *heads, dim, 32, seed=dim + 1, scale=0.125)
    made, at = [], 0
    for b, (e, n) in enumerate(zip(extends, c.lens)):
        q, k = far(gen, e, heads[0], n, heads[1], dim)
        k[:] = (k != 0) * 1536.0 if b % 2 else (k != 0) * -640.0
        v = torch.randn((n, heads[1], dim), generator=gen) + torch.arange(n)[:, None, None] * (4.0 / n)  # pieces differ
        made.append(fill(c, b, at, q, k.to(torch.bfloat16), v.to(torch.bfloat16)))
        at += e
    out, lse = c.run()
    for one, q, k, v in made:
        Exact(q, k, v, 0.125).check(out[one], lse[one])


@pytest.mark.parametrize("extends,prefixes,heads", BATCHES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("low", [False, True])
def test_values_near_the_largest(extends, prefixes, heads, dim, low):
    """Keys of low scores and values near the largest before keys of high scores and ordinary values, which are the result; and
    a rise over all keys."""
    gen = torch.Generator().manual_seed(dim + len(extends))
    c = Paged(extends, prefixes, *heads, dim, 16, seed=dim, scale=0.125)
    made, at = [], 0
    for b, (e, n) in enumerate(zip(extends, c.lens)):
        q, k = rising_scores(gen, e, heads[0], n, heads[1], dim, 60)
        v = huge(gen, n, heads[1], dim, most=100)
        if low:
            half = prefixes[b] * 2 // 3
            k[:half] = -k[:half].abs() - (k != 0)[:half] * 200.0
            v[:half], v[half:] = 2.0 ** 127, torch.randn(v[half:].shape, generator=gen).to(torch.bfloat16)
        made.append(fill(c, b, at, q, k, v))
        at += e
    out, lse = c.run()
    for one, q, k, v in made:
        Exact(q, k, v, 0.125).check(out[one], lse[one])
