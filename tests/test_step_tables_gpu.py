"""A step's tables built on the GPU from its requests' lengths: bit-exact against the oracle, and a step of an engine
with grouped heads run as a whole (tables, K/V rows stored at their slots, attention through the page table)."""

from __future__ import annotations

import random

import pytest
import torch

from minisgl_amd.core import Req
from minisgl_amd.kernel import lib
from minisgl_amd.kvcache import PagedTokenTable
from oracle import ref_gqa as R

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def make(cached, device, page_size, cols, seed, rows=None, spare=3):
    """A token table whose cached tokens lie on pages, and the free slots."""
    gen = torch.Generator().manual_seed(seed)
    held = [-(-c // page_size) for c in cached]
    need = sum(-(-d // page_size) for d in device)
    order = torch.randperm(need + spare, generator=gen).to(torch.int32) * page_size
    rows = len(cached) + 2 if rows is None else rows
    idx = torch.randperm(rows, generator=gen)[: len(cached)].tolist()
    table = torch.full((rows, cols), -1, dtype=torch.int32)
    at = 0
    for r, h in zip(idx, held):
        for j in range(h):
            n = min(page_size, cols - j * page_size)
            table[r, j * page_size : j * page_size + n] = order[at + j] + torch.arange(n, dtype=torch.int32)
        at += h
    return table, idx, order[at:].contiguous()


def run(table, idx, cached, device, free, page_size, alloc=None):
    dev_table = table.to(DEV)
    extends = [d - c for c, d in zip(cached, device)]
    t = lib.page_tables_from_lengths(dev_table, i32(idx), i32(cached), i32(device), free.to(DEV), page_size, max(device),
                                     max(extends), sum(extends), alloc)
    torch.cuda.synchronize()
    return dev_table.cpu(), t


def check(cached, device, page_size, cols, seed, alloc=None):
    table, idx, free = make(cached, device, page_size, cols, seed)
    got, t = run(table, idx, cached, device, free, page_size, alloc)
    ref = R.step_tables(table, idx, cached, device, free, page_size, -(-max(device) // page_size),
                        len(cached) if alloc is None else alloc)
    assert torch.equal(got, ref.token_table)
    assert torch.equal(t.page_table.cpu(), ref.page_table)
    assert t.out_loc.tolist() == ref.out_loc and t.positions.tolist() == ref.positions
    assert t.cu_seqlens_q.tolist() == ref.cu_seqlens_q and int(t.pages_taken) == ref.pages_taken


@pytest.mark.parametrize("page_size", [1, 3, 16, 64])
def test_ragged_step(page_size):
    r = random.Random(page_size)
    cached = [r.choice([0, 1, 15, 16, 17, 64, r.randint(0, 500)]) for _ in range(23)]
    device = [c + r.choice([0, 1, 1, 2, 47, 48, r.randint(1, 300)]) for c in cached]
    check(cached, device, page_size, 1000, seed=page_size)


@pytest.mark.parametrize("page_size", [1, 16])
def test_single_token_step_and_long_prompts(page_size):
    check([31, 32, 33, 0], [32, 33, 34, 1], page_size, 64, seed=1)
    check([0, 7, 4000], [5000, 4100, 4001], page_size, 5000, seed=2)


def test_many_requests():
    """More requests than a CTA has threads."""
    r = random.Random(3)
    cached = [r.randint(0, 40) for _ in range(700)]
    check(cached, [c + r.randint(0, 5) for c in cached], 8, 64, seed=3)


def test_last_page_is_cut_at_the_table_width():
    check([0, 90], [100, 100], 64, 100, seed=4)


def test_padding_takes_no_pages():
    """Requests past alloc_reqs read their rows as they are: a padded batch's dummy request, several times."""
    cached, device = [5, 0, 0, 0], [6, 40, 1, 1]
    table, idx, free = make(cached, device, 16, 64, seed=5)
    idx[3] = idx[2]
    table[idx[2]] = 16 * 7
    got, t = run(table, idx, cached, device, free, 16, alloc=2)
    ref = R.step_tables(table, idx, cached, device, free, 16, 3, 2)
    assert torch.equal(got, ref.token_table) and torch.equal(t.page_table.cpu(), ref.page_table)
    assert t.out_loc.tolist() == ref.out_loc and int(t.pages_taken) == ref.pages_taken == 3


def test_out_of_pages_writes_no_table():
    cached, device = [5, 0], [6, 400]
    table, idx, free = make(cached, device, 16, 512, seed=6)
    got, t = run(table, idx, cached, device, free[:24].contiguous(), 16)
    assert int(t.pages_taken) == 25 and torch.equal(got, table)
    assert t.cu_seqlens_q.tolist() == [0, 1, 401]


def test_sums_past_32_bits():
    """Lengths whose sums pass 2^31: the sums stop there and nothing is written outside the tables; pages that pass it are
    more than the free slots."""
    n, cols = 3000, 1 << 20
    table = torch.arange(cols, dtype=torch.int32, device=DEV).view(1, cols)
    same, zero, long = i32([0] * n), i32([0] * n), i32([cols] * n)
    t = lib.page_tables_from_lengths(table, same, zero, long, i32([]), 1, 100, 100, 1000, 0)
    cu = [min(i * cols, 2**31 - 1) for i in range(n + 1)]
    assert t.cu_seqlens_q.tolist() == cu and int(t.pages_taken) == 0
    assert t.out_loc[:100].tolist() == list(range(100)) and t.positions[:100].tolist() == list(range(100))
    assert torch.equal(t.page_table, torch.arange(100, dtype=torch.int32, device=DEV).expand(n, 100))
    t = lib.page_tables_from_lengths(table, same, zero, long, i32([7] * 100), 1, 100, 100, 1000)
    assert int(t.pages_taken) == 2**31 - 1 and t.cu_seqlens_q.tolist() == cu
    assert torch.equal(table[0], torch.arange(cols, dtype=torch.int32, device=DEV))
    # more new tokens than a table holds
    t = lib.page_tables_from_lengths(table, i32([0]), i32([0]), i32([cols]), i32([]), 1, 100, 2**31 - 1, 1000, 0)
    assert t.out_loc.tolist() == list(range(1000)) and t.cu_seqlens_q.tolist() == [0, cols]


def test_capture_and_replay():
    cached, device = [20, 3, 90], [21, 4, 91]
    table, idx, free = make(cached, device, 16, 128, seed=7, spare=10)
    dev, rows, c, d, f = table.to(DEV), i32(idx), i32(cached), i32(device), free.to(DEV)
    call = lambda: lib.page_tables_from_lengths(dev, rows, c, d, f, 16, 128, 1, 3)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        t = call()
    for step in range(4):
        now, then = [x + step for x in cached], [x + step for x in device]
        dev.copy_(table), c.copy_(i32(now)), d.copy_(i32(then))
        graph.replay()
        torch.cuda.synchronize()
        ref = R.step_tables(table, idx, now, then, free, 16, 8, 3)
        assert torch.equal(dev.cpu(), ref.token_table) and torch.equal(t.page_table.cpu(), ref.page_table)
        assert t.out_loc.tolist() == ref.out_loc and t.positions.tolist() == ref.positions


def test_paged_token_table_step_matches_allocate_paged():
    """The allocator's step on the device gives what its host-driven methods give, and runs out of pages as they do."""
    def fresh():
        return PagedTokenTable(40, 16, torch.zeros((6, 256), dtype=torch.int32, device=DEV))

    a, b = fresh(), fresh()
    for cached, device in (([0, 0, 0], [100, 3, 17]), ([100, 3, 17], [101, 40, 18])):
        reqs = [Req(table_idx=i, cached_len=c, device_len=d) for i, (c, d) in enumerate(zip(cached, device))]
        a.allocate_paged(reqs)
        t = b.allocate_step(reqs)
        assert torch.equal(a.page_table, b.page_table) and torch.equal(a.free_slots, b.free_slots)
        assert torch.equal(a.out_loc(reqs), t.out_loc)
        idx = i32([r.table_idx for r in reqs])
        whole = lib.page_table_from_tokens(a.page_table, idx, max(device), 16)
        for r, d in enumerate(device):
            assert torch.equal(whole[r, : -(-d // 16)], t.page_table[r, : -(-d // 16)])
    with pytest.raises(RuntimeError, match="out of KV pages"):
        b.allocate_step([Req(table_idx=4, cached_len=0, device_len=16 * 40)])
    assert torch.equal(a.free_slots, b.free_slots)


@pytest.mark.parametrize("page_size", [1, 16])
def test_steps_of_an_engine(page_size):
    """Prompts, then chunks on their prefixes, then single tokens: each step's tables, its K and V rows stored at their
    slots, and the attention over the pages, against the oracle on the tokens' own rows."""
    gen = torch.Generator().manual_seed(page_size)
    hq, hk, d, scale = 12, 2, 128, 0.1
    pages = 1200 // page_size
    table = PagedTokenTable(pages, page_size, torch.zeros((4, 512), dtype=torch.int32, device=DEV))
    pool_k, pool_v = (torch.full((pages, page_size, hk, d), float("nan"), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    history = [[torch.empty((0, hk, d), dtype=torch.bfloat16)] * 2 for _ in range(3)]
    lens = [0, 0, 0]
    for extends in ([150, 9, 64], [30, 140, 1], [1, 1, 1], [1, 1, 1]):
        reqs = [Req(table_idx=i, cached_len=n, device_len=n + e) for i, (n, e) in enumerate(zip(lens, extends))]
        T, first = sum(extends), all(n == 0 for n in lens)
        q, k, v = (torch.randn((T, h, d), generator=gen).to(torch.bfloat16) for h in (hq, hk, hk))
        qd, kd, vd = q.to(DEV), k.to(DEV), v.to(DEV)
        t = table.allocate_step(reqs)
        lib.store_rows(pool_k.view(-1, hk * d), t.out_loc, kd.view(T, hk * d))
        lib.store_rows(pool_v.view(-1, hk * d), t.out_loc, vd.view(T, hk * d))
        out, lse = torch.empty_like(qd), torch.empty((T, hq), device=DEV)
        lens = [n + e for n, e in zip(lens, extends)]
        if max(extends) == 1:
            lib.gqa_decode(qd, pool_k, pool_v, t.page_table, i32(lens), scale, out, lse)
        else:
            lib.gqa_chunk(qd, pool_k, pool_v, t.page_table, t.cu_seqlens_q, i32(lens), max(extends), scale, out, lse)
        refs, at = [], 0
        for b, e in enumerate(extends):
            history[b] = [torch.cat((h, x[at : at + e])) for h, x in zip(history[b], (k, v))]
            refs.append(R.attend(q[at : at + e], *history[b], scale))
            at += e
        ref = R.Attention(*(torch.cat(x) for x in zip(*refs)))
        assert ((out.double().cpu() - ref.out).abs() <= ref.out_bound).all()
        assert ((lse.double().cpu() - ref.lse).abs() <= ref.lse_bound).all()
        if first:  # whole prompts, without the cache: the same attention
            packed, packed_lse = torch.empty_like(qd), torch.empty((T, hq), device=DEV)
            lib.gqa_prompt(qd, kd, vd, t.cu_seqlens_q, scale, packed, packed_lse)
            assert ((packed.double().cpu() - ref.out).abs() <= ref.out_bound).all()
            assert ((packed_lse.double().cpu() - ref.lse).abs() <= ref.lse_bound).all()


def test_replays_with_fewer_and_more_new_tokens():
    """A captured step of padded size: fewer new tokens leave no slot of an earlier replay behind (nothing is stored at
    -1), none at all too; requests longer than the launch was made for, up to the tokens that the tables hold."""
    table, idx, free = make([20, 3, 90], [320, 303, 390], 16, 512, seed=8, spare=10)
    dev, rows, c, d, f = table.to(DEV), i32(idx), i32([0] * 3), i32([0] * 3), free.to(DEV)
    total = 64
    call = lambda: lib.page_tables_from_lengths(dev, rows, c, d, f, 16, 512, 4, total)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        t = call()
    rows_of_x = torch.ones((total, 8), dtype=torch.bfloat16, device=DEV)
    for extends in ([4, 4, 4], [1, 0, 2], [0, 0, 0], [4, 1, 4], [40, 4, 20], [0, 0, 300], [0, 1, 0]):
        now, then = [20, 3, 90], [20 + extends[0], 3 + extends[1], 90 + extends[2]]
        dev.copy_(table), c.copy_(i32(now)), d.copy_(i32(then))
        graph.replay()
        cache = torch.zeros((16 * 100, 8), dtype=torch.bfloat16, device=DEV)
        lib.store_rows(cache, t.out_loc, rows_of_x)
        torch.cuda.synchronize()
        ref = R.step_tables(table, idx, now, then, free, 16, 32, 3)
        n = min(sum(extends), total)
        assert torch.equal(dev.cpu(), ref.token_table) and torch.equal(t.page_table.cpu(), ref.page_table)
        assert t.out_loc.tolist() == ref.out_loc[:n] + [-1] * (total - n) and t.positions.tolist() == ref.positions[:n] + [0] * (total - n)
        assert t.cu_seqlens_q.tolist() == ref.cu_seqlens_q and int(t.pages_taken) == ref.pages_taken
        assert sorted(ref.out_loc[:n]) == cache[:, 0].nonzero().flatten().tolist()


@pytest.mark.parametrize("page_size", [1, 16, 24])
def test_out_of_pages_leaves_nothing_to_be_followed(page_size):
    """Kernels that are queued behind the tables find no slot and page 0, whatever the memory held."""
    cached, device = [5, 0, 70], [6, 3000, 75]
    table, idx, free = make(cached, device, page_size, 3000, seed=9)
    total = 3100
    for _ in range(3):
        torch.full((3 * 3000 + 2 * total + 5,), 77, dtype=torch.int32, device=DEV)  # given back at once
        dev = table.to(DEV)
        t = lib.page_tables_from_lengths(dev, i32(idx), i32(cached), i32(device), free[:2].to(DEV), page_size, 3000, 3000, total)
        torch.cuda.synchronize()
        assert torch.equal(dev.cpu(), table) and int(t.pages_taken) > 2 and t.cu_seqlens_q.tolist() == [0, 1, 3001, 3006]
        assert (t.page_table == 0).all() and (t.out_loc == -1).all() and (t.positions == 0).all()


@pytest.mark.parametrize("hint", [0, 1, 5, 10 ** 6])
def test_most_new_tokens_only_size_the_launch(hint):
    cached, device = [0, 17, 4000, 3], [2500, 18, 4100, 3]
    table, idx, free = make(cached, device, 16, 4500, seed=10)
    dev = table.to(DEV)
    t = lib.page_tables_from_lengths(dev, i32(idx), i32(cached), i32(device), free.to(DEV), 16, 4100, hint, 2601)
    ref = R.step_tables(table, idx, cached, device, free, 16, 257, 4)
    assert torch.equal(dev.cpu(), ref.token_table) and torch.equal(t.page_table.cpu(), ref.page_table)
    assert t.out_loc.tolist() == ref.out_loc and t.positions.tolist() == ref.positions
