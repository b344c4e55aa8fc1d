"""The 4-bit cache on the GPU: rows in and out bit by bit against the 64-bit oracle, and attention over it within the bounds
that oracle/ref_gqa.py derives (its kernels multiply the codes' values, exact in bf16, and round as the bf16 ones do)."""

from __future__ import annotations

import random

import pytest
import torch

from minisgl_amd.kernel import lib
from oracle import ref_gqa as R
from oracle import ref_mx4 as M

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
NAN = float("nan")


def randn(gen, *shape):
    return torch.randn(shape, generator=gen).to(torch.bfloat16)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def cumulative(x):
    out = [0]
    for v in x:
        out.append(out[-1] + v)
    return out


def pool_of(codes, scales, by_head):
    """The tensors on the GPU, with a head's rows of a page next to each other or a token's heads."""
    if not by_head:
        return lib.MX4Pool(codes.to(DEV).contiguous(), scales.to(DEV).contiguous())
    pool = lib.mx4_pool(*codes.shape[:3], 2 * codes.shape[3], DEV)
    pool.codes.copy_(codes)
    pool.scales.copy_(scales)
    return pool


def special_rows(dim):
    """Blocks of zeros, subnormals, the largest and smallest values, ties and borders of every code, infinities and NaN."""
    blocks = [torch.zeros(32), -torch.zeros(32), torch.full((32,), 3.3895e38), torch.full((32,), -2.0 ** -133), torch.full((32,), 2.0 ** -126)]
    for e in (-126, -125, -124, -130, -20, 0, 3, 60, 125):  # of the block's largest, 4 or 7.96875 units
        for top in (1.0, 1.9921875):
            borders = torch.tensor([0.0, 0.25, 0.25390625, 0.75, 0.74609375, 1.25, 1.2578125, 1.75, 1.7421875, 2.5, 2.515625, 3.5, 3.484375, 5.0, 5.03125, 6.0])
            blocks.append(torch.cat((torch.tensor([top * 4]), borders[1:], -borders)) * 2.0 ** (e - 2))
    for bad in (float("inf"), -float("inf"), NAN):
        b = torch.ones(32)
        b[17] = bad
        blocks.append(b)
    while len(blocks) % (dim // 32):
        blocks.append(torch.ones(32))
    return torch.stack(blocks).to(torch.bfloat16).view(-1, 1, dim)


@pytest.mark.parametrize("by_head", [False, True])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page_size", [1, 4, 64])
def test_store_bits(dim, page_size, by_head):
    gen = torch.Generator().manual_seed(dim + page_size)
    heads = 3
    special = special_rows(dim).expand(-1, heads, dim)
    k = torch.cat((randn(gen, 50, heads, dim), special, randn(gen, 7, heads, dim) * 1e-30))
    v = torch.cat((special, randn(gen, 57, heads, dim) * 1e20))
    T = k.shape[0]
    pages = -(-T // page_size) + 2
    slots = torch.randperm(pages * page_size, generator=gen)[:T]
    pools = []
    for x in (k, v):
        codes = torch.randint(0, 256, (pages, page_size, heads, dim // 2), generator=gen, dtype=torch.uint8)
        scales = torch.randint(0, 256, (pages, page_size, heads, dim // 32), generator=gen, dtype=torch.uint8)
        pools.append((codes, scales, pool_of(codes, scales, by_head)))
    skipped = torch.tensor([5, 60])
    given = slots.clone()
    given[skipped] = torch.tensor([-1, pages * page_size])
    for dtype in (torch.int32, torch.int64):
        lib.mx4_store(pools[0][2], pools[1][2], given.to(DEV, dtype), k.to(DEV), v.to(DEV))
    kept = torch.ones(T, dtype=torch.bool)
    kept[skipped] = False
    for x, (codes, scales, pool) in zip((k, v), pools):
        c, s = M.rounded(x)
        codes.view(-1, heads, dim // 2)[slots[kept]] = c[kept]
        scales.view(-1, heads, dim // 32)[slots[kept]] = s[kept]
        assert torch.equal(pool.scales.cpu(), scales)
        assert torch.equal(pool.codes.cpu(), codes)
    # and back: what the codes stand for, exactly
    k_back, v_back = lib.mx4_load(pools[0][2], pools[1][2], given.to(DEV))
    for back, (codes, scales, _) in zip((k_back, v_back), pools):
        want = M.values(codes.view(-1, heads, dim // 2)[slots], scales.view(-1, heads, dim // 32)[slots])
        want[skipped] = 0.0
        torch.testing.assert_close(back.cpu().double(), want.to(torch.bfloat16).double(), rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("dim", [64, 128])
def test_every_code_and_scale(dim):
    """Rows of every byte of codes under every scale; those past bf16's range are infinities."""
    codes = torch.arange(256, dtype=torch.uint8).view(-1, 1, 16).expand(16, 256, 16).reshape(-1, 16)[:, None].repeat(1, 1, dim // 32)
    scales = torch.arange(256, dtype=torch.uint8).repeat_interleave(16)[:, None, None].expand(-1, 1, dim // 32)
    codes, scales = codes[:, None], scales[:, None]  # pages of one token
    pool = pool_of(codes, scales, False)
    k, v = lib.mx4_load(pool, pool, torch.arange(codes.shape[0], device=DEV))
    want = M.values(codes, scales)[:, 0].to(torch.bfloat16)
    torch.testing.assert_close(k.cpu(), want, rtol=0, atol=0, equal_nan=True)
    torch.testing.assert_close(v.cpu(), want, rtol=0, atol=0, equal_nan=True)


def test_store_strided():
    """Rows that are parts of a projection's output, into a part of a larger pool, and out into strided rows; no rows at all."""
    gen = torch.Generator().manual_seed(4)
    T, heads, dim, page = 21, 2, 128, 8
    qkv = randn(gen, T, 6 * dim).to(DEV)
    k, v = qkv[:, 2 * dim : 4 * dim].unflatten(1, (heads, dim)), qkv[:, 4 * dim :].unflatten(1, (heads, dim))
    codes = torch.zeros((10, page, heads + 1, dim // 2), dtype=torch.uint8, device=DEV)
    scales = torch.zeros((10, page, heads + 1, dim // 32), dtype=torch.uint8, device=DEV)
    part = lib.MX4Pool(codes[3:, :, 1:], scales[3:, :, 1:])
    other = lib.mx4_pool(7, page, heads, dim, DEV)
    slots = torch.randperm(7 * page, generator=gen)[:T].to(DEV)
    lib.mx4_store(part, other, slots, k, v)
    assert not codes[:3].any() and not codes[:, :, 0].any() and not scales[:3].any() and not scales[:, :, 0].any()
    out = torch.full((heads, T, dim + 8), NAN, dtype=torch.bfloat16, device=DEV)
    k_back, v_back = lib.mx4_load(part, other, slots, k=out[:, :, :dim].transpose(0, 1))
    assert k_back.data_ptr() == out.data_ptr() and out[:, :, dim:].isnan().all()
    assert torch.equal(k_back.cpu().double(), M.values(*M.rounded(k.cpu())))
    assert torch.equal(v_back.cpu().double(), M.values(*M.rounded(v.cpu())))
    before = codes.clone()
    lib.mx4_store(part, other, slots[:0], k[:0], v[:0])
    assert lib.mx4_load(part, other, slots[:0])[0].shape == (0, heads, dim) and torch.equal(codes, before)


# ---- attention


def check(out, lse, ref, what=""):
    out, lse = out.double().cpu(), lse.double().cpu()
    assert not out.isnan().any() and not lse.isnan().any() and torch.equal(torch.isinf(lse), torch.isinf(ref.lse)), what
    over = (out - ref.out).abs() - ref.out_bound
    assert over.max() <= 0, f"{what}: out is {over.max():.3e} past its bound"
    off = torch.where(ref.lse.isinf(), 0.0, lse - ref.lse).abs() - ref.lse_bound
    assert off.max() <= 0, f"{what}: lse is {off.max():.3e} past its bound"


class Paged:
    """A batch over pools that are NaN in every row that no request owns, and past every length."""

    def __init__(self, extends, prefixes, q_heads, kv_heads, dim, page_size, seed, spare_rows=0, scale=None, by_head=True):
        gen = torch.Generator().manual_seed(seed)
        self.extends, self.lens, self.by_head = list(extends), [e + p for e, p in zip(extends, prefixes)], by_head
        self.scale = dim ** -0.5 if scale is None else scale
        need = [-(-n // page_size) for n in self.lens]
        pages = sum(need) + 3
        order = torch.randperm(pages, generator=gen).to(torch.int32)
        shape = (pages, page_size, kv_heads)
        self.k, self.v = ((torch.full((*shape, dim // 2), 0x77, dtype=torch.uint8), torch.full((*shape, dim // 32), 255, dtype=torch.uint8)) for _ in "kv")
        self.pt = torch.full((len(need), max(max(need), 1)), -7, dtype=torch.int32)  # unused entries are no pages
        self.page_size, at = page_size, 0
        for b, (n, L) in enumerate(zip(need, self.lens)):
            self.pt[b, :n] = order[at : at + n]
            at += n
            for pool in (self.k, self.v):
                self.put(pool, b, range(L), randn(gen, L, kv_heads, dim))
        self.T = sum(self.extends)
        self.q = randn(gen, self.T + spare_rows, q_heads, dim)

    def row(self, b, j):
        return int(self.pt[b, j // self.page_size]) * self.page_size + j % self.page_size

    def put(self, pool, b, keys, x):
        rows = torch.tensor([self.row(b, j) for j in keys], dtype=torch.long)
        for whole, some in zip(pool, M.rounded(x)):
            whole.view(-1, *whole.shape[2:])[rows] = some

    def ref(self):
        """The bounds of oracle/ref_gqa.py are for sums within fp32's normal range. A numerator below it, 2^-126, may come out as
        anything up to twice itself, and so may its product with a value: at most L of each, over a sum of numerators that is at
        least 1 (the largest's), bring 2^-126 L (max |v| + 1) to a result."""
        v = M.values(*self.v)
        ref = R.chunk(self.q, M.values(*self.k), v, self.pt, self.extends, self.lens, self.scale)
        return ref._replace(out_bound=ref.out_bound + 2.0 ** -126 * max(self.lens) * (v.nan_to_num(posinf=0.0, neginf=0.0).abs().max() + 1))

    def run(self, max_q=None, workspace=None, total_keys=-1, decode=False):
        q = self.q.to(DEV)
        out = torch.full_like(q, NAN)
        lse = torch.full(q.shape[:2], NAN, device=DEV)
        k, v = pool_of(*self.k, self.by_head), pool_of(*self.v, self.by_head)
        total = sum(self.lens) if total_keys == -1 else total_keys
        if decode:
            lib.gqa_decode_mx4(q, k, v, self.pt.to(DEV), i32(self.lens), self.scale, out, lse, workspace, total)
        else:
            lib.gqa_chunk_mx4(q, k, v, self.pt.to(DEV), i32(cumulative(self.extends)), i32(self.lens),
                              max(self.extends) if max_q is None else max_q, self.scale, out, lse, workspace, total)
        torch.cuda.synchronize()
        return out, lse


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads", [(1, 1), (8, 1), (4, 4), (14, 2), (16, 1), (20, 1), (33, 1), (64, 1), (80, 1), (48, 3)])
def test_decode_heads(dim, heads):
    c = Paged([1] * 5, [0, 31, 32, 200, 777], *heads, dim, 16, heads[0] + dim)
    check(*c.run(decode=True), c.ref())


@pytest.mark.parametrize("by_head", [False, True])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page_size", [1, 2, 8, 16, 32, 64, 256])
def test_decode_pages(dim, page_size, by_head):
    c = Paged([1] * 7, [0, 1, 62, 63, 64, 300, 1999], 8, 2, dim, page_size, page_size + dim, by_head=by_head)
    check(*c.run(decode=True), c.ref())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens", [[20000], [9000, 3, 70, 5000], [40] * 40 + [6000] * 3, [1500] * 130])
def test_decode_split(dim, lens):
    c = Paged([1] * len(lens), [n - 1 for n in lens], 4, 2, dim, 64, len(lens))
    check(*c.run(decode=True), c.ref())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("most", [3200, 3500])
def test_many_keys_in_one_piece_or_not(dim, most):
    """Either side of the most keys that as many CTAs as compute units take in one piece."""
    lens = [most, 1, 33, 0, 255, 256, 257, 2900] + [(37 * i) % 700 for i in range(22)]
    c = Paged([1] * 30, [n - 1 for n in lens], 16, 8, dim, 16, most)
    check(*c.run(decode=True), c.ref())
    c = Paged([2, 1, 5] * 10, lens, 16, 8, dim, 16, most)
    check(*c.run(), c.ref())


@pytest.mark.parametrize("batch,kv_heads,group,most,extend", [
    (24, 8, 8, 500, 6),     # more CTAs of 16 rows than compute units, up to 1000 keys
    (24, 8, 8, 1300, 6),    # and past it
    (70, 8, 8, 200, 6),     # more than run at once, up to 256 keys
    (40, 8, 8, 150, 12),    # of fuller requests
    (20, 2, 4, 120, 3),     # up to 256 keys in one piece: four waves
    (40, 8, 4, 1700, 1),    # one piece of more CTAs than run at once
    (40, 8, 4, 2100, 1),    # cut
    (40, 8, 8, 3000, 5),    # 32 rows, in one piece
    (40, 8, 8, 4200, 5)])   # cut
def test_every_choice(batch, kv_heads, group, most, extend):
    gen = torch.Generator().manual_seed(batch + most)
    extends = torch.randint(1, extend + 1, (batch,), generator=gen).tolist()
    prefixes = [most] + torch.randint(0, 200, (batch - 1,), generator=gen).tolist()
    extends[-1] = extend
    c = Paged(extends, prefixes, kv_heads * group, kv_heads, 64, 16, most)
    check(*c.run(), c.ref())


def test_decode_without_keys():
    c = Paged([1] * 4, [9, -1, 33, -1], 4, 2, 128, 16, 3)
    out, lse = c.run(decode=True)
    check(out, lse, c.ref())
    assert (out[1] == 0).all() and (lse[3] == -float("inf")).all()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads", [(4, 4), (8, 2), (14, 2), (16, 1)])
@pytest.mark.parametrize("extends,prefixes", [
    ([1, 2, 3, 4], [10, 0, 700, 31]),
    ([5, 0, 1, 40, 17], [100, 50, 0, 0, 1500]),
    ([130, 64, 1], [0, 1000, 64]),
    ([300], [33]),
])
def test_chunk(dim, heads, extends, prefixes):
    c = Paged(extends, prefixes, *heads, dim, 16, sum(extends) + dim, spare_rows=5)
    out, lse = c.run()
    check(out[: c.T], lse[: c.T], c.ref())
    assert out[c.T :].isnan().all() and lse[c.T :].isnan().all()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("total", [-1, None])
def test_chunk_long(dim, total):
    """Enough rows for the values to be laid out first, with pages of one token; memory by the sum of lengths or by the table."""
    c = Paged([700, 1, 333, 0, 64], [100, 900, 0, 5, 700], 16, 4, dim, 1, 5 + dim)
    check(*c.run(total_keys=total), c.ref())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("extends,prefixes,heads", [
    ([256], [600], (64, 8)),           # streamed: blocks would be few
    ([256], [3900], (64, 8)),          # laid out: long
    ([530], [40], (32, 4)),            # laid out: more
    ([160, 3, 0, 300], [9, 2000, 30, 0], (16, 4))])
def test_more_rows_streamed_or_laid_out(extends, prefixes, heads, dim):
    c = Paged(extends, prefixes, *heads, dim, 16, dim + len(extends))
    check(*c.run(), c.ref())


def test_chunk_many_requests():
    r = random.Random(6)
    extends = [r.choice([0, 1, 2, 17, 70]) for _ in range(140)]
    c = Paged(extends, [r.choice([0, 3, 64, 130]) for _ in extends], 12, 3, 64, 4, 6)
    check(*c.run(), c.ref())


def test_chunk_rows_without_keys():
    """Fewer keys than queries: the first queries attend none."""
    c = Paged([5, 90], [-3, -60], 8, 2, 128, 4, 8)
    check(*c.run(), c.ref())


@pytest.mark.parametrize("extends,prefixes", [([3], [40]), ([40], [20]), ([200], [10]), ([9], [3000])])
@pytest.mark.parametrize("dim", [64, 128])
def test_nan_reaches_rows_that_attend_it(dim, extends, prefixes):
    """A block of a value or key that is NaN, at a token inside the chunk: rows before it are as without it, rows from it on are
    NaN, of a value only in the block's dims."""
    at = prefixes[0] + extends[0] // 2  # the token
    for what in "vk":
        c = Paged(extends, prefixes, 4, 2, dim, 16, 11)
        ref = c.ref()
        getattr(c, what)[1].view(-1, 2, dim // 32)[c.row(0, at), 1, 1] = 255  # head 1, second block
        out, lse = c.run()
        out, lse = out.double().cpu(), lse.double().cpu()
        hit = torch.zeros(out.shape, dtype=torch.bool)
        hit[extends[0] // 2 :, 2:, 32:64 if what == "v" else dim] = True
        if what == "k":
            hit[extends[0] // 2 :, 2:] = True
        assert torch.equal(out.isnan(), hit), what
        assert torch.equal(lse.isnan(), hit.any(-1) if what == "k" else torch.zeros(lse.shape, dtype=torch.bool)), what
        over = torch.where(hit, 0.0, (out - ref.out).abs() - ref.out_bound)
        assert over.max() <= 0, what


@pytest.mark.parametrize("extends,prefixes", [([1, 1], [3000, 70]), ([3, 20], [200, 100]), ([140], [1000])])
@pytest.mark.parametrize("dim", [64, 128])
def test_largest_values(dim, extends, prefixes):
    """Sums on the way to a result pass fp32's range unless the numerators leave room."""
    c = Paged(extends, prefixes, 4, 2, dim, 16, 12, scale=2.0 ** -30)  # weights alike
    c.v[0].fill_(0x77)  # 6 and 6
    c.v[1].fill_(252)
    out, lse = c.run()
    want = torch.tensor(6 * 2.0 ** 125, dtype=torch.float64)
    # 2^-8 for the numerators and for the result
    assert ((out.double().cpu() - want).abs() <= 2.02 * 2.0 ** -8 * want).all()
    assert ((lse.double().cpu() - c.ref().lse).abs() <= c.ref().lse_bound + 2.0 ** -19).all()  # a sum of 24 and more, rounded


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("order", ["falling", "rising"])
def test_values_of_every_size(dim, order):
    """Blocks from next to the largest to the smallest that a result can hold, by token: in tiles before and after one another."""
    c = Paged([1, 40], [700, 300], 4, 2, dim, 32, 14, scale=1.0)
    gen = torch.Generator().manual_seed(15)
    for b, L in enumerate(c.lens):
        for j in range(L):
            e = 122 - (240 * j) // L if order == "falling" else -118 + (240 * j) // L
            c.put(c.v, b, [j], (torch.randn((1, 2, dim), generator=gen).clamp(-8, 8) * 2.0 ** e).to(torch.bfloat16))
    check(*c.run(), c.ref())


@pytest.mark.parametrize("size", [2.0 ** -120, 2.0 ** -60, 2.0 ** 60, 2.0 ** 120])
def test_values_of_a_size(size):
    c = Paged([1, 9], [2000, 100], 8, 2, 128, 64, 16)
    gen = torch.Generator().manual_seed(17)
    for b, L in enumerate(c.lens):
        c.put(c.v, b, range(L), (torch.randn((L, 2, 128), generator=gen).clamp(-8, 8) * size).to(torch.bfloat16))
    check(*c.run(), c.ref())


def test_pages_and_lengths_outside():
    """Page ids outside the pool are taken as its first and last page, lengths past the page table as its width, and queries past
    total_q are left out: what the arrays hold is never followed out of the tensors."""
    c = Paged([1, 1, 1], [90, 40, 20], 4, 2, 128, 32, 18)
    pages = c.pt.shape[1]
    c.v[0].copy_(torch.randint(0, 256, c.v[0].shape, generator=torch.Generator().manual_seed(1), dtype=torch.uint8))
    c.k[1].fill_(126)
    c.v[1].fill_(127)
    c.pt[0, 1], c.pt[1, 0], c.pt[2, 0] = 1 << 30, -(1 << 31), c.k[0].shape[0]
    given = list(c.lens)
    c.lens[2] = 1 << 30
    c.pt[2, 1:] = -1
    out, lse = c.run(decode=True, total_keys=1000)
    c.pt.clamp_(0, c.k[0].shape[0] - 1)
    c.lens = given[:2] + [pages * 32]
    check(out, lse, c.ref())


@pytest.mark.parametrize("scale", [1e-6, 3.0, 100.0])
def test_scales(scale):
    c = Paged([1, 3, 2], [500, 64, 2000], 8, 2, 128, 16, 13, scale=scale)
    check(*c.run(), c.ref())


def test_past_32_bits():
    """Pools of more than 4 GiB, tokens at their ends."""
    pages, ps, heads, dim = 140_000, 64, 8, 128
    k, v = lib.mx4_pool(pages, ps, heads, dim, DEV), lib.mx4_pool(pages, ps, heads, dim, DEV)
    assert k.codes.numel() > 1 << 32
    gen = torch.Generator().manual_seed(1)
    L = 150
    pt = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32)
    j = torch.arange(L)
    slots = pt[0].long()[j // ps] * ps + j % ps
    x, y, q = randn(gen, L, heads, dim), randn(gen, L, heads, dim), randn(gen, 1, heads, dim)
    lib.mx4_store(k, v, slots.to(DEV), x.to(DEV), y.to(DEV))
    kb, vb = lib.mx4_load(k, v, slots.to(DEV, torch.int32))
    assert torch.equal(kb.cpu().double(), M.values(*M.rounded(x))) and torch.equal(vb.cpu().double(), M.values(*M.rounded(y)))
    out, lse = torch.empty_like(q, device=DEV), torch.empty((1, heads), device=DEV)
    lib.gqa_decode_mx4(q.to(DEV), k, v, pt.to(DEV), i32([L]), dim ** -0.5, out, lse)
    ref = R.attend(q, M.values(*M.rounded(x)), M.values(*M.rounded(y)), dim ** -0.5)
    check(out, lse, ref)


# ---- streams, graphs, workspaces


@pytest.mark.parametrize("decode", [True, False])
def test_another_stream(decode):
    """Without a workspace, on a stream that is not the current one, behind what that stream does."""
    c = Paged([1] * 3 if decode else [150, 3, 60], [5000, 10, 900], 8, 2, 128, 16, 21)
    ref = c.ref()
    q = c.q.to(DEV)
    k, v, pt, lens, cu = pool_of(*c.k, True), pool_of(*c.v, True), c.pt.to(DEV), i32(c.lens), i32(cumulative(c.extends))
    out, lse = torch.full_like(q, NAN), torch.full(q.shape[:2], NAN, device=DEV)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        late = torch.zeros_like(q)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.cuda._sleep(1_000_000)
            late.copy_(q)
        if decode:
            lib.gqa_decode_mx4(late, k, v, pt, lens, c.scale, out, lse, stream=side)
        else:
            lib.gqa_chunk_mx4(late, k, v, pt, cu, lens, max(c.extends), c.scale, out, lse, stream=side)
        torch.full((1 << 20,), NAN, device=DEV)  # what the current stream allocates meanwhile
        side.synchronize()
        check(out, lse, ref)


def test_rows_on_another_stream():
    """In and out on a stream that is not the current one, results made for it, alone or beside a given one."""
    gen = torch.Generator().manual_seed(26)
    T, heads, dim = 500, 4, 128
    x, y = randn(gen, T, heads, dim), randn(gen, T, heads, dim)
    want = [M.values(*M.rounded(z)).to(torch.bfloat16) for z in (x, y)]
    pools = [lib.mx4_pool(40, 16, heads, dim, DEV) for _ in "kv"]
    slots = torch.randperm(640, generator=gen)[:T].to(DEV)
    side, xd, yd = torch.cuda.Stream(), x.to(DEV), y.to(DEV)
    torch.cuda.synchronize()
    for given in (False, True):
        late = torch.zeros_like(xd)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.cuda._sleep(1_000_000)
            late.copy_(xd)
        lib.mx4_store(*pools, slots, late, yd, stream=side)
        k = torch.zeros_like(xd) if given else None
        side.wait_stream(torch.cuda.current_stream())
        k, v = lib.mx4_load(*pools, slots, k=k, stream=side)
        torch.full((1 << 20,), NAN, device=DEV)
        side.synchronize()
        assert torch.equal(k.cpu(), want[0]) and torch.equal(v.cpu(), want[1])
        for p in pools:
            p.codes.zero_()
        torch.cuda.synchronize()


def test_rows_captured():
    """Stores and loads in a graph follow what their tensors hold at each replay; slots of -1 are skipped."""
    gen = torch.Generator().manual_seed(27)
    T, heads, dim = 33, 2, 64
    pools = [lib.mx4_pool(5, 16, heads, dim, DEV) for _ in "kv"]
    x, y = (torch.zeros((T, heads, dim), dtype=torch.bfloat16, device=DEV) for _ in "kv")
    k, v = torch.empty_like(x), torch.empty_like(x)
    slots = torch.arange(T, dtype=torch.int32, device=DEV)

    def call():
        lib.mx4_store(*pools, slots, x, y)
        lib.mx4_load(*pools, slots, k, v)

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for new in (33, 20, 33):
        a, b = randn(gen, T, heads, dim), randn(gen, T, heads, dim)
        s = torch.randperm(80, generator=gen)[:T].int()
        s[new:] = -1
        x.copy_(a), y.copy_(b), slots.copy_(s)
        graph.replay()
        torch.cuda.synchronize()
        for got, z in ((k, a), (v, b)):
            want = M.values(*M.rounded(z)).to(torch.bfloat16)
            want[new:] = 0
            assert torch.equal(got.cpu(), want)


def test_tensors_that_do_not_fit():
    x = torch.zeros((2, 4, 128), dtype=torch.bfloat16, device=DEV)
    p = lib.mx4_pool(2, 4, 4, 128, DEV)
    i = torch.zeros(2, dtype=torch.int32, device=DEV)
    half = lib.mx4_pool(2, 4, 2, 128, DEV)
    refused = [
        (lambda: lib.mx4_store(p, half, i, x, x), "same shape"), (lambda: lib.mx4_store(p, p, i, x[:, :2], x), "k must be"),
        (lambda: lib.mx4_store(p, p, i, x, x.float()), "v must be"), (lambda: lib.mx4_store(p, p, i.float(), x, x), "indices must be"),
        (lambda: lib.mx4_store(p, p, i[:1], x, x), "k must be"), (lambda: lib.mx4_store(lib.MX4Pool(p.codes, p.scales[..., :3]), p, i, x, x), "for each 32 dims"),
        (lambda: lib.mx4_store(lib.MX4Pool(p.codes.int(), p.scales), p, i, x, x), "uint8"),
        (lambda: lib.gqa_decode_mx4(x[..., :64], p, p, i.view(2, 1), i, 0.1, x[..., :64]), "q's D"),
        (lambda: lib.gqa_decode_mx4(x[:, :3].contiguous(), p, p, i.view(2, 1), i, 0.1, x[:, :3].contiguous()), "heads that divide"),
        (lambda: lib.gqa_decode_mx4(x, p, p, i.view(2, 1), i[:1], 0.1, x), "one token"), (lambda: lib.gqa_decode_mx4(x, p, p, i, i, 0.1, x), "page_table"),
        (lambda: lib.gqa_chunk_mx4(x, p, p, i.view(2, 1), i, i, 1, 0.1, x), "cu_seqlens_q"),
        (lambda: lib.gqa_chunk_mx4(x, p, p, i.view(2, 1), None, i, 1, 0.1, x), "cu_seqlens_q"),
    ]
    for call, text in refused:
        with pytest.raises(AssertionError, match=text):
            call()
    other = lib.MX4Pool(torch.zeros((2, 4, 4, 64), dtype=torch.uint8, device=DEV), torch.zeros((2, 4, 4, 4), dtype=torch.uint8, device=DEV))
    with pytest.raises(lib.MLAKernelError, match="same strides"):
        lib.gqa_decode_mx4(x, p, other, i.view(2, 1), i, 0.1, torch.empty_like(x))
    with pytest.raises(lib.MLAKernelError, match="overlap"):
        lib.mx4_load(p, p, i, k=x[:1].expand(2, 4, 128))


@pytest.mark.parametrize("decode", [True, False])
def test_captured(decode):
    """Two graphs with workspaces of their own, replayed by turns with eager calls between, following their lengths."""
    cases = [Paged([1] * 3 if decode else [150, 3, 60], [5000, 10, 900], 8, 2, 128, 16, s) for s in (22, 23)]
    runs = []
    for c in cases:
        q, k, v, pt, cu = c.q.to(DEV), pool_of(*c.k, True), pool_of(*c.v, True), c.pt.to(DEV), i32(cumulative(c.extends))
        lens, out, lse = i32(c.lens), torch.full_like(c.q, NAN, device=DEV), torch.full(c.q.shape[:2], NAN, device=DEV)
        total = pt.numel() * 16
        n = lib.gqa_mx4_workspace_bytes(1 if decode else 150, 8, 2, 128, 3, pt.shape[1] * 16, total)
        ws = torch.empty(n, dtype=torch.uint8, device=DEV)

        def call(q=q, k=k, v=v, pt=pt, cu=cu, lens=lens, out=out, lse=lse, ws=ws, c=c, total=total):
            if decode:
                lib.gqa_decode_mx4(q, k, v, pt, lens, c.scale, out, lse, ws, total)
            else:
                lib.gqa_chunk_mx4(q, k, v, pt, cu, lens, 150, c.scale, out, lse, ws, total)

        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        runs.append((c, graph, lens, out, lse, call))
    for shift in (0, 700, 100, 0):
        for c, graph, lens, out, lse, call in runs:
            c.lens = [max(n - shift, e) for n, e in zip(c.lens_at_start, c.extends)] if hasattr(c, "lens_at_start") else c.lens
            c.lens_at_start = getattr(c, "lens_at_start", list(c.lens))
            lens.copy_(i32(c.lens))
            out.fill_(NAN)
            graph.replay()
            torch.cuda.synchronize()
            ref = c.ref()
            check(out, lse, ref, f"replay, {shift} fewer")
            got = out.clone()
            call()
            torch.cuda.synchronize()
            assert torch.equal(got, out)


def test_same_results_every_time():
    c = Paged([1, 1, 30], [9000, 50, 4000], 8, 2, 128, 16, 24)
    first = c.run()
    for _ in range(3):
        again = c.run()
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_workspace_is_enough():
    """A workspace of the size asked for, with other bytes around it left as they are; one byte less is refused."""
    c = Paged([70, 3], [2000, 10], 8, 2, 128, 16, 25)
    n = lib.gqa_mx4_workspace_bytes(70, 8, 2, 128, 2, c.pt.shape[1] * 16, sum(c.lens))
    block = torch.full((n + 4096,), 0x5A, dtype=torch.uint8, device=DEV)
    check(*c.run(workspace=block[2048 : 2048 + n]), c.ref())
    assert (block[:2048] == 0x5A).all() and (block[2048 + n :] == 0x5A).all()
    with pytest.raises(lib.MLAKernelError, match="workspace"):
        c.run(workspace=block[2048 : 2047 + n])


def test_a_step():
    """A step as an engine runs it: the tables of its requests, norms and rotation from the projection's output, rows into the
    4-bit cache, attention; then the next step's token."""
    from minisgl_amd.core import Req
    from minisgl_amd.kvcache import PagedTokenTable

    gen = torch.Generator().manual_seed(31)
    hq, hk, d, ps, eps = 8, 2, 128, 16, 1e-6
    table = PagedTokenTable(64, ps, torch.zeros((9, 512), dtype=torch.int32, device=DEV))
    k_pool, v_pool = lib.mx4_pool(64, ps, hk, d, DEV), lib.mx4_pool(64, ps, hk, d, DEV)
    angle = torch.arange(512)[:, None] * 0.02 ** (torch.arange(d // 2) / (d // 2))
    cos_sin = torch.cat((angle.cos(), angle.sin()), 1).float()
    qw, kw = randn(gen, d), randn(gen, d)
    reqs = [Req(3, 0, 90), Req(1, 0, 33), Req(7, 0, 1)]
    keys, vals = [[], [], []], [[], [], []]
    for step in range(3):
        T = sum(r.extend_len for r in reqs)
        qkv = randn(gen, T, (hq + 2 * hk) * d)
        t = table.allocate_step(reqs)
        dev = qkv.to(DEV)
        q, k, v = (x.unflatten(1, (-1, d)) for x in dev.split([hq * d, hk * d, hk * d], 1))
        lib.qk_norm_rope(q, k, v, qw.to(DEV), kw.to(DEV), eps, t.positions, cos_sin.to(DEV), False, q, k, v)
        lib.mx4_store(k_pool, v_pool, t.out_loc, k, v)
        out, lse = torch.empty((T, hq, d), dtype=torch.bfloat16, device=DEV), torch.empty((T, hq), device=DEV)
        lens = i32([r.device_len for r in reqs])
        lib.gqa_chunk_mx4(q, k_pool, v_pool, t.page_table, t.cu_seqlens_q, lens, max(r.extend_len for r in reqs), d ** -0.5, out, lse,
                          total_keys=sum(r.device_len for r in reqs))
        torch.cuda.synchronize()
        # the rotated rows against the oracle, and the rest from the rows as they were rounded
        raw_q, raw_k, raw_v = (x.unflatten(1, (-1, d)) for x in qkv.split([hq * d, hk * d, hk * d], 1))
        for got, raw, w in ((q, raw_q, qw), (k, raw_k, kw)):
            want, bound = M.norm_rope(raw, w, eps, t.positions.cpu(), cos_sin, False)
            assert ((got.cpu().double() - want).abs() <= bound).all()
        assert torch.equal(v.cpu(), raw_v)
        at = 0
        for i, r in enumerate(reqs):
            rows = slice(at, at + r.extend_len)
            keys[i].append(M.values(*M.rounded(k[rows].cpu())))
            vals[i].append(M.values(*M.rounded(v[rows].cpu())))
            check(out[rows], lse[rows], R.attend(q[rows].cpu(), torch.cat(keys[i]), torch.cat(vals[i]), d ** -0.5), f"step {step}, request {i}")
            at += r.extend_len
            r.complete_one()
