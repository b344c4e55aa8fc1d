"""Views that the grouped-head attention and the step's tables take as they are: pools whose K and V lie side by side,
single pages, tokens, heads and rows, whose strides torch gives any value."""

from __future__ import annotations

import pytest
import torch

from minisgl_amd.kernel import lib
from oracle import ref_gqa as R
from test_gqa_gpu import DEV, check, i32, randn

pytestmark = pytest.mark.gpu


def one_of_many(t, dim, n=3, pad=5):
    """``t`` (size 1 in ``dim``) as a view whose stride there is no multiple of anything."""
    strides = list(t.stride())
    strides[dim] = 7 * t.numel() + pad
    got = t.as_strided(t.shape, strides)
    assert got.stride(dim) == strides[dim] and torch.equal(got, t)
    return got


@pytest.mark.parametrize("decode", [True, False])
def test_pool_of_single_tokens_with_k_and_v_side_by_side(decode):
    gen = torch.Generator().manual_seed(1)
    rows, hq, hk, d = 700, 8, 2, 128
    both = randn(gen, rows, 2, hk, d)
    dev = both.to(DEV)
    extends, lens = ([1, 1], [300, 41]) if decode else ([70, 3], [300, 41])
    pt = torch.randperm(rows, generator=gen)[: 2 * 300].view(2, 300).to(torch.int32)
    q = randn(gen, sum(extends), hq, d)
    ref = R.chunk(q, both[:, 0][:, None], both[:, 1][:, None], pt, extends, lens, 0.1)
    out, lse = torch.empty_like(q, device=DEV), torch.empty((sum(extends), hq), device=DEV)
    k, v = dev[:, 0].unsqueeze(1), dev[:, 1].unsqueeze(1)
    assert k.stride(0) == 2 * hk * d
    if decode:
        lib.gqa_decode(q.to(DEV), k, v, pt.to(DEV), i32(lens), 0.1, out, lse)
    else:
        lib.gqa_chunk(q.to(DEV), k, v, pt.to(DEV), i32([0, 70, 73]), i32(lens), 70, 0.1, out, lse)
    check(out, lse, ref)


def test_one_page_one_request_one_head():
    gen = torch.Generator().manual_seed(2)
    k, v, q = randn(gen, 1, 64, 1, 64), randn(gen, 1, 64, 1, 64), randn(gen, 1, 1, 64)
    pt, lens = torch.zeros((1, 1), dtype=torch.int32), [50]
    ref = R.chunk(q, k, v, pt, [1], lens, 0.2)
    kd, vd = (one_of_many(one_of_many(x.to(DEV), 0), 2) for x in (k, v))
    qd, out = (one_of_many(one_of_many(x, 0), 1) for x in (q.to(DEV), torch.empty_like(q, device=DEV)))
    lse = one_of_many(torch.empty((1, 1), device=DEV), 1)
    lib.gqa_decode(qd, kd, vd, one_of_many(one_of_many(pt.to(DEV), 0), 1), i32(lens), 0.2, out, lse)
    check(out, lse, ref)


def test_prompt_of_one_token_and_one_kv_head():
    gen = torch.Generator().manual_seed(3)
    for T in (1, 40):
        q, k, v = randn(gen, T, 4, 64), randn(gen, T, 1, 64), randn(gen, T, 1, 64)
        kd, vd = (one_of_many(x.to(DEV), 1) for x in (k, v))
        qd, out = q.to(DEV), torch.empty_like(q, device=DEV)
        if T == 1:
            qd, out, kd, vd = (one_of_many(x, 0) for x in (qd, out, kd, vd))
        lse = torch.empty((T, 4), device=DEV)
        lib.gqa_prompt(qd, kd, vd, i32([0, T]), 0.2, out, lse)
        check(out, lse, R.prompt(q, k, v, [T], 0.2))


def test_token_table_of_one_row():
    row = torch.zeros((1, 100), dtype=torch.int32, device=DEV)
    table = row.as_strided((1, 100), (3, 1))
    t = lib.page_tables_from_lengths(table, i32([0]), i32([0]), i32([40]), i32([16, 64, 0]), 16, 40, 40, 40)
    ref = R.step_tables(torch.zeros((1, 100), dtype=torch.int32), [0], [0], [40], torch.tensor([16, 64, 0]), 16, 3, 1)
    assert torch.equal(row.cpu(), ref.token_table) and torch.equal(t.page_table.cpu(), ref.page_table) and t.out_loc.tolist() == ref.out_loc


def test_pages_that_do_not_follow_one_another_are_refused():
    pool = torch.zeros((6, 2, 16, 2, 64), dtype=torch.bfloat16, device=DEV)
    q, out = torch.zeros((1, 4, 64), dtype=torch.bfloat16, device=DEV), torch.zeros((1, 4, 64), dtype=torch.bfloat16, device=DEV)
    with pytest.raises(AssertionError, match="follow one another"):
        lib.gqa_decode(q, pool[:, 0], pool[:, 1], i32([[0, 1]]), i32([20]), 0.1, out)


def test_expanded_tensors():
    """Rows that lie on each other: read where only read (one query, one KV head for all), refused where an entry past
    the memory would be, and where results would be written over each other."""
    gen = torch.Generator().manual_seed(4)
    T, hq, hk, d = 40, 4, 2, 64
    q, k, v = randn(gen, 1, hq, d), randn(gen, T, 1, d), randn(gen, T, 1, d)
    qd, kd, vd = q.to(DEV).expand(T, hq, d), k.to(DEV).expand(T, hk, d), v.to(DEV).expand(T, hk, d)
    out, lse = torch.empty((T, hq, d), dtype=torch.bfloat16, device=DEV), torch.empty((T, hq), device=DEV)
    lib.gqa_prompt(qd, kd, vd, i32([0, T]), 0.2, out, lse)
    check(out, lse, R.prompt(q.expand(T, hq, d), k.expand(T, hk, d), v.expand(T, hk, d), [T], 0.2))
    with pytest.raises(AssertionError, match="contiguous"):
        lib.gqa_prompt(qd, kd, vd, i32([0, T]), 0.2, out, torch.empty((T, 1), device=DEV).expand(T, hq))
    with pytest.raises(lib.MLAKernelError, match="lse_stride"):
        lib.gqa_prompt(qd, kd, vd, i32([0, T]), 0.2, out, torch.empty((1, hq), device=DEV).expand(T, hq))
    with pytest.raises(lib.MLAKernelError, match="out strides"):
        lib.gqa_prompt(qd, kd, vd, i32([0, T]), 0.2, torch.empty_like(out[:1]).expand(T, hq, d))
    pool, one = torch.zeros((6, 16, hk, d), dtype=torch.bfloat16, device=DEV), i32([[3], [3]])
    with pytest.raises(AssertionError, match="page_table is int32"):
        lib.gqa_decode(qd[:2], pool, pool, one.expand(2, 4), i32([20, 30]), 0.1, out[:2])
    with pytest.raises(lib.MLAKernelError, match="pt_stride"):
        lib.gqa_decode(qd[:2], pool, pool, i32([[0, 1, 2, 3]]).expand(2, 4), i32([20, 30]), 0.1, out[:2])
    with pytest.raises(AssertionError, match="token_table is int32"):
        lib.page_tables_from_lengths(one.expand(2, 64), i32([0, 1]), i32([0, 0]), i32([20, 20]), i32(list(range(0, 96, 16))), 16, 20, 20, 40)
    with pytest.raises(lib.MLAKernelError, match="token table"):
        lib.page_tables_from_lengths(i32([[0] * 64]).expand(2, 64), i32([0, 1]), i32([0, 0]), i32([20, 20]), i32(list(range(0, 96, 16))), 16, 20, 20, 40)
