"""Calls on a stream that is not the current one: memory that a call takes from torch's allocator is taken on the call's
stream. A block that the current stream has just given back may still be written by work queued there, and nothing orders
another stream's launch behind that work."""

from __future__ import annotations

import pytest
import torch

from minisgl_amd.kernel import lib
from oracle import ref_gqa as R

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def freed_while_written(nbytes):
    """A block of ``nbytes`` that the current stream gives back with writes to it still queued; its address."""
    block = torch.empty((nbytes,), dtype=torch.uint8, device=DEV)
    for _ in range(300):
        block.fill_(0x7F)
    return block.data_ptr()


def owned_by(stream, nbytes):
    """Whether the allocator holds memory of ``stream`` for a block of ``nbytes``."""
    return any(s["stream"] == stream.cuda_stream and s["total_size"] >= nbytes for s in torch.cuda.memory_snapshot())


@pytest.mark.parametrize("decode", [True, False])
def test_attention_without_a_workspace_on_another_stream(decode):
    gen = torch.Generator().manual_seed(1)
    randn = lambda *shape: torch.randn(shape, generator=gen).to(torch.bfloat16)  # noqa: E731
    lens, ps, hq, hk, d = [4000, 2500], 16, 8, 1, 128
    extends = [1, 1] if decode else [3, 2]
    pages = [-(-n // ps) for n in lens]
    k, v, q = randn(sum(pages), ps, hk, d), randn(sum(pages), ps, hk, d), randn(sum(extends), hq, d)
    pt = torch.zeros((2, max(pages)), dtype=torch.int32)
    pt[0, : pages[0]], pt[1, : pages[1]] = torch.arange(pages[0]), torch.arange(pages[0], sum(pages))
    ref = R.chunk(q, k, v, pt, extends, lens, 0.1)
    dev = [x.to(DEV) for x in (q, k, v, pt)]
    cu, dl = i32([0, extends[0], sum(extends)]), i32(lens)
    nbytes = lib.gqa_workspace_bytes(max(extends), hq, hk, d)
    for side in (torch.cuda.Stream(), torch.cuda.Stream()):
        out, lse = torch.zeros_like(dev[0]), torch.zeros((sum(extends), hq), device=DEV)
        torch.cuda.synchronize()
        freed_while_written(nbytes)
        if decode:
            lib.gqa_decode(*dev, dl, 0.1, out, lse, stream=side)
        else:
            lib.gqa_chunk(*dev, cu, dl, max(extends), 0.1, out, lse, stream=side)
        torch.cuda.synchronize()
        assert owned_by(side, nbytes)
        assert ((out.double().cpu() - ref.out).abs() <= ref.out_bound).all()
        assert ((lse.double().cpu() - ref.lse).abs() <= ref.lse_bound).all()


def test_tables_on_another_stream():
    gen = torch.Generator().manual_seed(2)
    n, ps, cols = 256, 16, 4096
    cached = torch.randint(0, 500, (n,), generator=gen).tolist()
    lens = [c + 1 + i % 700 for i, c in enumerate(cached)]
    total, width = sum(b - a for a, b in zip(cached, lens)), -(-max(lens) // ps)
    table = torch.zeros((n, cols), dtype=torch.int32)
    free = torch.randperm(sum(-(-x // ps) for x in lens), generator=gen).to(torch.int32) * ps
    ref = R.step_tables(table, range(n), cached, lens, free, ps, width, n)
    args = i32(list(range(n))), i32(cached), i32(lens), free.to(DEV)
    nbytes = 4 * (n * width + 2 * total + n + 2)
    for side in (torch.cuda.Stream(), torch.cuda.Stream()):
        dev = table.to(DEV)
        torch.cuda.synchronize()
        at = freed_while_written(nbytes)
        t = lib.page_tables_from_lengths(dev, *args, ps, max(lens), max(b - a for a, b in zip(cached, lens)), total, stream=side)
        assert t.page_table.untyped_storage().data_ptr() != at
        torch.cuda.synchronize()
        assert owned_by(side, nbytes)
        assert torch.equal(t.page_table.cpu(), ref.page_table) and torch.equal(dev.cpu(), ref.token_table)
        assert t.out_loc.tolist() == ref.out_loc and t.positions.tolist() == ref.positions
        assert t.cu_seqlens_q.tolist() == ref.cu_seqlens_q and int(t.pages_taken) == ref.pages_taken


def test_tables_used_where_they_were_asked_for():
    """The tables belong to the call's stream; freed while the caller's stream still reads them, their memory is kept."""
    side = torch.cuda.Stream()
    table, free = torch.zeros((64, 4096), dtype=torch.int32, device=DEV), i32(list(range(0, 64 * 4096, 16)))
    rows, zero, lens = i32(list(range(64))), i32([0] * 64), i32([4096] * 64)
    call = lambda: lib.page_tables_from_lengths(table, rows, zero, lens, free, 16, 4096, 4096, 64 * 4096, stream=side)  # noqa: E731
    torch.cuda.synchronize()
    want = None
    for _ in range(4):
        t = call()
        torch.cuda.current_stream().wait_stream(side)
        junk = torch.empty((1 << 26,), device=DEV)
        for _ in range(200):
            junk.fill_(1.0)
        got = t.out_loc.clone()
        at = t.page_table.untyped_storage().data_ptr()
        del t
        with torch.cuda.stream(side):
            other = torch.full((64 * 256 + 2 * 64 * 4096 + 66,), -5, dtype=torch.int32, device=DEV)
        assert other.data_ptr() != at
        torch.cuda.synchronize()
        want = got if want is None else want
        assert torch.equal(got, want) and int(got.min()) >= 0
        del other, junk


def test_capture_on_a_forked_stream():
    """A captured call on a stream forked from the capturing one, without a workspace; replays between eager calls."""
    gen = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(s, generator=gen).to(torch.bfloat16) for s in ((1, 8, 128), (200, 16, 1, 128), (200, 16, 1, 128)))
    pt = torch.arange(200, dtype=torch.int32)[None]
    ref = R.chunk(q, k, v, pt, [1], [3100], 0.1)
    dev, dl = [x.to(DEV) for x in (q, k, v, pt)], i32([3100])
    out, lse, side = torch.zeros_like(dev[0]), torch.zeros((1, 8), device=DEV), torch.cuda.Stream()
    lib.gqa_decode(*dev, dl, 0.1, out, lse)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        now = torch.cuda.current_stream()
        side.wait_stream(now)
        lib.gqa_decode(*dev, dl, 0.1, out, lse, stream=side)
        now.wait_stream(side)
    for _ in range(4):
        out.fill_(float("nan")), lse.fill_(float("nan"))
        graph.replay()
        junk = torch.full((1 << 24,), float("nan"), device=DEV)
        other, other_lse = torch.empty_like(out), torch.empty_like(lse)
        lib.gqa_decode(*dev, dl, 0.1, other, other_lse)
        torch.cuda.synchronize()
        assert torch.equal(out, other) and torch.equal(lse, other_lse)
        assert ((out.double().cpu() - ref.out).abs() <= ref.out_bound).all()
        del junk


def test_other_results_on_another_stream():
    """The calls that make their result, where none is given, and rows that are copied to be stored."""
    gen = torch.Generator().manual_seed(4)
    T, side = 3001, torch.cuda.Stream()
    qkv = torch.randn((T, 512 + 576), generator=gen).to(torch.bfloat16).to(DEV)
    w512, w576 = torch.ones(512, dtype=torch.bfloat16, device=DEV), torch.ones(576, dtype=torch.bfloat16, device=DEV)
    pos, cos_sin = i32(list(range(T))), torch.randn((T, 64), generator=gen).to(DEV)
    table, rows = i32(list(range(64 * 4096))).view(64, 4096), i32(list(range(64)))
    wide, slots = qkv.view(T, 2, 544).transpose(0, 1).contiguous().transpose(0, 1), i32(list(range(T)))

    def store(stream=None):
        cache = torch.zeros((T, 1088), dtype=torch.bfloat16, device=DEV)
        torch.cuda.synchronize()
        freed_while_written(T * 1088 * 2)
        lib.store_rows(cache, slots, wide, stream=stream)
        return cache

    calls = [
        (T * 576 * 2, lambda **kw: lib.rmsnorm(qkv[:, :576], w576, 1e-6, **kw)),
        (T * 576 * 2, lambda **kw: lib.latent_rows(qkv[:, 512:], w512, pos, cos_sin, 1e-6, False, **kw)),
        (T * 576 * 2, lambda **kw: lib.qkv_a_rows(qkv.clone() if not kw else copy, 512, w512, w512, pos, cos_sin, 1e-6, False, **kw)),
        (64 * 256 * 4, lambda **kw: lib.page_table_from_tokens(table, rows, 4096, 16, **kw)),
        (T * 1088 * 2, store),
    ]
    for nbytes, call in calls:
        copy = qkv.clone()
        want = call()
        torch.cuda.synchronize()
        at = freed_while_written(nbytes)
        got = call(stream=side)
        assert call is store or got.untyped_storage().data_ptr() != at
        torch.cuda.synchronize()
        assert owned_by(side, nbytes) and torch.equal(got, want)


def test_tables_captured_on_a_forked_stream():
    table, free = torch.zeros((4, 256), dtype=torch.int32, device=DEV), i32(list(range(0, 16 * 64, 16)))
    rows, cached, lens, side = i32([0, 1, 2, 3]), i32([0] * 4), i32([100, 3, 17, 256]), torch.cuda.Stream()
    call = lambda **kw: lib.page_tables_from_lengths(table, rows, cached, lens, free, 16, 256, 256, 400, **kw)  # noqa: E731
    want = [x.clone() for x in call()]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        now = torch.cuda.current_stream()
        side.wait_stream(now)
        t = call(stream=side)
        now.wait_stream(side)
        copy = t.out_loc + 0
    for _ in range(4):
        table.zero_()
        graph.replay()
        junk = torch.full((1 << 22,), -9, dtype=torch.int32, device=DEV)
        eager = call()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) and torch.equal(c, b) for a, b, c in zip(t, want, eager)) and torch.equal(copy, want[1])
        del junk
