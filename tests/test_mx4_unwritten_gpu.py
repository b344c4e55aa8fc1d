"""The 4-bit cache's attention beside values that pass bf16's range (scales 253 and 254, which random bytes have too): in rows that
nobody attends or ever wrote, and at tokens that some rows of a chunk attend."""

from __future__ import annotations

import pytest
import torch

from minisgl_amd.kernel import lib
from oracle import ref_gqa as R
from oracle import ref_mx4 as M
from test_mx4_gpu import DEV, Paged, check, i32, randn

pytestmark = pytest.mark.gpu

# of unowned rows: codes and scales, None for random bytes
GARBAGE = [(0x77, 253), (0xFF, 254), (0x44, 254), (None, None), (0x77, 255)]


def spoil(c, codes, scales):
    """Every row that no request owns."""
    gen = torch.Generator().manual_seed(5)
    rest = torch.ones(c.k[0].shape[0] * c.page_size, dtype=torch.bool)
    for b, n in enumerate(c.lens):
        rest[[c.row(b, j) for j in range(n)]] = False
    for pool in (c.k, c.v):
        for x, byte in zip(pool, (codes, scales)):
            flat = x.view(-1, *x.shape[2:])
            flat[rest] = torch.randint(0, 256, flat[rest].shape, generator=gen, dtype=torch.uint8) if byte is None else byte


@pytest.mark.parametrize("by_head", [False, True])
@pytest.mark.parametrize("page_size", [1, 16, 32, 64, 256])
@pytest.mark.parametrize("extends,prefixes,heads", [
    ([1] * 6, [0, 30, 32, 99, 700, 3000], (8, 2)),  # single tokens, short and in pieces
    ([1] * 3, [5, 40, 1300], (16, 1)),
    ([3, 20, 1], [200, 77, 0], (8, 2)),             # chunks: 16 rows, and 32
    ([7, 2], [2500, 300], (16, 4)),
    ([9, 70], [30, 1000], (16, 4)),
    ([300, 1], [33, 40], (8, 2))])
def test_rows_that_nobody_attends(extends, prefixes, heads, page_size, by_head):
    for dim in (64, 128):
        c = Paged(extends, prefixes, *heads, dim, page_size, page_size + dim, by_head=by_head)
        ref = c.ref()
        for garbage in GARBAGE:
            spoil(c, *garbage)
            check(*c.run(decode=max(extends) == 1), ref, f"head_dim {dim}, unowned rows {garbage}")


@pytest.mark.parametrize("page_size", [16, 64])
def test_rows_that_nobody_attends_of_values_laid_out(page_size):
    c = Paged([700, 1, 333, 64], [100, 900, 5, 700], 16, 4, 128, page_size, 9)
    ref = c.ref()
    for garbage in GARBAGE[::3]:
        spoil(c, *garbage)
        check(*c.run(), ref, f"unowned rows {garbage}")


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page_size", [32, 64])
def test_new_pool_in_used_memory(dim, page_size):
    """A pool of memory with other bytes, a prompt stored to it, and its next token."""
    gen = torch.Generator().manual_seed(page_size)
    L, hq, hk = 75, 8, 2
    pages = -(-L // page_size)
    k, v = lib.mx4_pool(pages, page_size, hk, dim, DEV), lib.mx4_pool(pages, page_size, hk, dim, DEV)
    for p in (k, v):  # as the allocator may give it
        p.codes.fill_(0x77), p.scales.fill_(253)
    x, y, q = randn(gen, L, hk, dim), randn(gen, L, hk, dim), randn(gen, 1, hq, dim)
    lib.mx4_store(k, v, torch.arange(L, device=DEV), x.to(DEV), y.to(DEV))
    out, lse = torch.empty_like(q, device=DEV), torch.empty((1, hq), device=DEV)
    lib.gqa_decode_mx4(q.to(DEV), k, v, i32([list(range(pages))]), i32([L]), dim ** -0.5, out, lse)
    check(out, lse, R.attend(q, M.values(*M.rounded(x)), M.values(*M.rounded(y)), dim ** -0.5))


@pytest.mark.parametrize("extends,prefixes,heads", [
    ([1], [40], (4, 2)), ([3], [40], (4, 2)), ([40], [20], (4, 2)), ([9], [3000], (4, 2)), ([5, 20], [100, 31], (16, 4)), ([300], [33], (8, 2)),
    ([700, 333, 64], [5, 0, 400], (16, 4))])  # the last: laid out
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page_size", [16, 64])
@pytest.mark.parametrize("scale", [253, 254])
def test_infinities_reach_rows_that_attend_them(scale, page_size, dim, extends, prefixes, heads):
    """A block of V at a token inside a chunk with every code under one of the two scales: rows before the token are as
    without it; from it on, dims that pass bf16's range are not finite, and all others within their bounds."""
    c = Paged(extends, prefixes, *heads, dim, page_size, 11)
    b = len(extends) - 1
    first = extends[b] // 2
    row, head, block = c.row(b, prefixes[b] + first), heads[1] - 1, 1
    codes, scales = (x.view(-1, *x.shape[2:]) for x in c.v)
    order = torch.randperm(32, generator=torch.Generator().manual_seed(3)) % 16
    mine = slice(16 * block, 16 * block + 16)
    codes[row, head, mine] = 0
    without = c.ref()  # the block's values 0
    code = torch.where(M.ELEMENTS[order].abs() * 2.0 ** (scale - 127) < 2.0 ** 128, order, 0)
    codes[row, head, mine] = (code[0::2] + 16 * code[1::2]).to(torch.uint8)
    scales[row, head, block] = scale
    finite = c.ref()  # those in the range
    codes[row, head, mine] = (order[0::2] + 16 * order[1::2]).to(torch.uint8)
    out, lse = (x.double().cpu() for x in c.run())

    start = sum(extends[:b])
    hit = torch.zeros(out.shape, dtype=torch.bool)  # rows, heads and dims of the block
    G = heads[0] // heads[1]
    hit[start + first : c.T, G * head : G * head + G, 32 * block : 32 * block + 32] = True
    past = torch.zeros(dim, dtype=torch.bool)
    past[32 * block : 32 * block + 32] = code != order
    past = hit & past
    assert past.any() and not out[past].isfinite().any()
    for where, ref in ((~hit, without), (hit & ~past, finite)):
        over = (out - ref.out).abs()[where] - ref.out_bound[where]
        assert over.max() <= 0, f"{over.max():.3e} past its bound"
    assert ((lse - without.lse).abs() <= without.lse_bound).all()
