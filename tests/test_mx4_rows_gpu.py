"""Rows into the 4-bit cache: as many as a launch holds."""

from __future__ import annotations

import pytest
import torch

from minisgl_amd.kernel import lib
from oracle import ref_mx4 as M
from test_mx4_gpu import DEV

pytestmark = pytest.mark.gpu


def test_store_of_more_than_two_to_the_31_pieces():
    """A thread a piece of 8 dims, of K and V: 2^24 rows of 8 heads of 128 and some, nearly all of them skipped. Row t is the 128
    values from the 8 t-th on, and every head's."""
    T, heads, dim, ps = (1 << 24) + 37, 8, 128, 16
    assert 1 << 31 < T * heads * (dim // 8) < (1 << 32) - 256
    gen = torch.Generator(device=DEV).manual_seed(1)
    flat = torch.randn((8 * T + dim,), generator=gen, device=DEV, dtype=torch.bfloat16)
    k = flat.as_strided((T, heads, dim), (8, 0, 1))
    v = flat.flip(0).as_strided((T, heads, dim), (8, 0, 1))
    stored = [0, 1, 255, 4096, (1 << 23) + 3, (1 << 24) - 1, 1 << 24, T - 1]
    indices = torch.full((T,), -1, dtype=torch.int32, device=DEV)
    at = torch.tensor(stored, device=DEV)
    indices[at] = torch.arange(len(stored), dtype=torch.int32, device=DEV) * 3
    pools = [lib.mx4_pool(2, ps, heads, dim, DEV) for _ in "kv"]
    for p in pools:
        p.codes.fill_(0x5A), p.scales.fill_(0x5A)
    lib.mx4_store(*pools, indices, k, v)
    for p, x in zip(pools, (k, v)):
        codes, scales = p.codes.cpu().flatten(0, 1), p.scales.cpu().flatten(0, 1)
        want = M.rounded(x[at].cpu())
        mine = torch.arange(len(stored)) * 3
        assert torch.equal(codes[mine], want[0]) and torch.equal(scales[mine], want[1])
        rest = torch.ones(2 * ps, dtype=torch.bool)
        rest[mine] = False
        assert (codes[rest] == 0x5A).all() and (scales[rest] == 0x5A).all()
