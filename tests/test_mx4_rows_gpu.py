"""Rows into the 4-bit cache: as many as a launch holds, and pools of every order of their dimensions."""

from __future__ import annotations

import itertools

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


@pytest.mark.parametrize("order", itertools.permutations(range(3)))
@pytest.mark.parametrize("room", [0, 1])
def test_pools_of_every_order(order, room):
    """Pages, tokens and heads with strides in any order, with and without room between them; codes and scales not alike."""
    gen = torch.Generator().manual_seed(2)
    pages, ps, heads, dim = 3, 8, 2, 64

    def part(width, order):
        sizes = [(pages, ps, heads)[i] + room for i in order]
        made = torch.full((*sizes, width), 0x5A, dtype=torch.uint8, device=DEV)
        return made.permute(*(order.index(i) for i in range(3)), 3)[:pages, :ps, :heads]

    pools = [lib.MX4Pool(part(dim // 2, order), part(dim // 32, o)) for o in (order[::-1], order)]
    slots = torch.randperm(pages * ps, generator=gen)
    x, y = (torch.randn((pages * ps, heads, dim), generator=gen).to(torch.bfloat16) for _ in "kv")
    lib.mx4_store(*pools, slots.to(DEV), x.to(DEV), y.to(DEV))
    for p, z in zip(pools, (x, y)):
        codes, scales = M.rounded(z)
        assert torch.equal(p.codes.cpu().flatten(0, 1)[slots], codes) and torch.equal(p.scales.cpu().flatten(0, 1)[slots], scales)
    k, v = lib.mx4_load(*pools, slots.to(DEV))
    assert torch.equal(k.cpu().double(), M.values(*M.rounded(x))) and torch.equal(v.cpu().double(), M.values(*M.rounded(y)))
