"""Refusals of the grouped-head attention and step-table entry points, all made on the host before anything is
launched (so the device pointers here need not be any), the workspace's size, and the oracle's own checks."""

from __future__ import annotations

import ctypes

import pytest
import torch

from minisgl_amd.kernel import lib
from minisgl_amd.core import Req
from minisgl_amd.kvcache import PagedTokenTable
from oracle import ref_gqa as R

P = 1 << 20  # a 16-byte aligned address, never followed
OK, INVALID, UNSUPPORTED = 0, 1, 3


def prompt(**kw):
    a = dict(q=P, qt=1024, qh=128, k=P, kr=256, kh=128, v=P, vr=256, vh=128, cu=P, batch=0, T=10, hq=8, hk=2, d=128, scale=0.1,
             out=P, ot=1024, oh=128, lse=P, lt=8, stream=None)
    assert set(kw) <= set(a)
    a.update({"batch": 2, **kw})
    return lib.load_library().mla_gqa_prompt_bf16(*a.values())


def chunk(**kw):
    a = dict(q=P, qt=1024, qh=128, k=P, kr=256, kh=128, v=P, vr=256, vh=128, pages=10, ps=16, pt=P, cols=4, pts=4, cu=P, lens=P,
             batch=2, T=10, max_q=8, hq=8, hk=2, d=128, scale=0.1, ws=P, ws_bytes=1 << 40, out=P, ot=1024, oh=128, lse=P,
             lt=8, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.load_library().mla_gqa_chunk_bf16(*a.values())


def decode(**kw):
    a = dict(q=P, qt=1024, qh=128, k=P, kr=256, kh=128, v=P, vr=256, vh=128, pages=10, ps=16, pt=P, cols=4, pts=4, lens=P,
             batch=2, hq=8, hk=2, d=128, scale=0.1, ws=P, ws_bytes=1 << 40, out=P, ot=1024, oh=128, lse=P, lt=8, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.load_library().mla_gqa_decode_bf16(*a.values())


def tables(**kw):
    a = dict(tt=P, rows=8, cols=64, stride=64, idx=P, cached=P, device=P, batch=2, alloc=2, free=P, num_free=5, ps=16,
             max_extend=9, pt=P, pt_cols=4, pts=4, loc=P, pos=P, new=12, cu=P, taken=P, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.load_library().mla_page_tables_from_lengths(*a.values())


ATTENTION = [
    (dict(hq=8, hk=3), INVALID, "no multiple"), (dict(hq=0), INVALID, "no multiple"), (dict(hk=0), INVALID, "no multiple"),
    (dict(d=96), UNSUPPORTED, "head_dim"), (dict(d=256), UNSUPPORTED, "head_dim"), (dict(batch=-1), INVALID, "batch"),
    (dict(q=None), INVALID, "null"), (dict(k=None), INVALID, "null"), (dict(v=None), INVALID, "null"), (dict(out=None), INVALID, "null"),
    (dict(q=P + 8), INVALID, "aligned"), (dict(k=P + 2), INVALID, "aligned"), (dict(v=P + 8), INVALID, "aligned"), (dict(out=P + 4), INVALID, "aligned"),
    (dict(qt=1028), INVALID, "q strides"), (dict(qh=-128), INVALID, "q strides"),
    (dict(kr=1 << 32), UNSUPPORTED, "4 GiB"), (dict(kr=260), INVALID, "k and v strides"), (dict(kh=4), INVALID, "k and v strides"), (dict(vr=-256), INVALID, "k and v strides"),
    (dict(oh=124), INVALID, "out strides"), (dict(ot=1022), INVALID, "out strides"), (dict(ot=1020), INVALID, "out strides"),
    (dict(hq=8192, hk=1), UNSUPPORTED, "query heads"), (dict(lt=7), INVALID, "lse_stride"), (dict(scale=0.0), INVALID, "scale"), (dict(scale=float("nan")), INVALID, "scale"),
    (dict(scale=float("inf")), INVALID, "scale"),
]
PAGED = [
    (dict(ps=24), UNSUPPORTED, "page_size"), (dict(ps=0), UNSUPPORTED, "page_size"), (dict(pages=0), INVALID, "num_pages"),
    (dict(pages=1 << 20, ps=1 << 12), UNSUPPORTED, "2^31 rows"), (dict(batch=70000), UNSUPPORTED, "65535"), (dict(cols=0), INVALID, "pt_cols"), (dict(pts=3), INVALID, "pt_stride"), (dict(pt=None), INVALID, "null"), (dict(lens=None), INVALID, "null"),
    (dict(ws=None), INVALID, "null"), (dict(ws=P + 8), INVALID, "workspace"), (dict(ws_bytes=1000), INVALID, "workspace"),
]


@pytest.mark.parametrize("call,cases", [(prompt, ATTENTION + [(dict(cu=None), INVALID, "null"), (dict(T=-1), INVALID, "total_q")]),
                                        (chunk, ATTENTION + PAGED + [(dict(cu=None), INVALID, "null"), (dict(max_q=-1), INVALID, "max_q")]),
                                        (decode, ATTENTION + PAGED)])
def test_attention_refusals(call, cases):
    for kw, code, text in cases:
        rc, message = call(**kw), lib.load_library().mla_last_error().decode()
        assert rc == code and text in message, (kw, rc, message)


def test_empty_batches_are_calls_that_do_nothing():
    assert prompt(batch=0) == prompt(T=0) == chunk(batch=0) == chunk(T=0) == chunk(max_q=0) == decode(batch=0) == OK


def test_table_refusals():
    for kw, text in ((dict(batch=0), "batch"), (dict(batch=70000), "batch"), (dict(alloc=3), "alloc_reqs"), (dict(alloc=-1), "alloc_reqs"),
                     (dict(num_free=-1), "num_free"), (dict(ps=0), "page_size"), (dict(tt=None), "null"), (dict(free=None), "null"),
                     (dict(idx=None), "null"), (dict(loc=None), "null"), (dict(cu=None), "null"), (dict(taken=None), "null"),
                     (dict(rows=0), "token table"), (dict(stride=63), "token table"), (dict(pts=3), "pt_stride"), (dict(new=-1), "total_new"),
                     (dict(max_extend=-1), "max_extend"), (dict(pt=None), "null")):
        assert tables(**kw) == INVALID and text in lib.load_library().mla_last_error().decode(), kw


def test_workspace_bytes():
    """Fixed by the rows of a request alone; refusals as the calls'."""
    assert lib.gqa_workspace_bytes(1, 8, 1, 128) == lib.gqa_workspace_bytes(2, 64, 8, 128)
    sizes = [lib.gqa_workspace_bytes(n, 8, 1, 128) for n in (1, 4, 8)]
    assert sizes == sorted(sizes) and all(s % 16 == 0 and 0 < s < 1 << 30 for s in sizes + [lib.gqa_workspace_bytes(4096, 64, 8, 64)])
    with pytest.raises(lib.MLAKernelError, match="head_dim"):
        lib.gqa_workspace_bytes(1, 8, 1, 80)
    with pytest.raises(lib.MLAKernelError, match="no multiple"):
        lib.gqa_workspace_bytes(1, 8, 5, 128)
    assert lib.load_library().mla_gqa_workspace_bytes(1, 8, 1, 128, None) == INVALID
    n = ctypes.c_int64(0)
    assert lib.load_library().mla_gqa_workspace_bytes(-1, 8, 1, 128, ctypes.byref(n)) == INVALID


def test_workspace_of_many_queries_is_enough_for_fewer():
    sizes = [lib.gqa_workspace_bytes(n, 8, 1, 128) for n in (0, 1, 2, 3, 4, 5, 8, 9, 16, 17, 300, 4096)]
    assert sizes == sorted(sizes)


def test_no_workspace_where_keys_are_split():
    for rc in (chunk(cols=1000, pts=1000, ws=None, ws_bytes=0), decode(cols=1000, pts=1000, ws=None, ws_bytes=0)):
        assert rc == INVALID and "workspace" in lib.load_library().mla_last_error().decode()


def test_bindings_refuse_host_tensors_and_wrong_types():
    q, k = torch.zeros((4, 8, 64), dtype=torch.bfloat16), torch.zeros((4, 2, 64), dtype=torch.bfloat16)
    cu, pool, pt = torch.zeros(2, dtype=torch.int32), torch.zeros((3, 16, 2, 64), dtype=torch.bfloat16), torch.zeros((1, 2), dtype=torch.int32)
    with pytest.raises(AssertionError, match="GPU"):
        lib.gqa_prompt(q, k, k, cu, 0.1, torch.empty_like(q))
    with pytest.raises(AssertionError, match="GPU"):
        lib.gqa_decode(q[:1], pool, pool, pt, cu[:1], 0.1, torch.empty_like(q[:1]))
    with pytest.raises(AssertionError, match="GPU"):
        lib.page_tables_from_lengths(pt, cu[:1], cu[:1], cu[:1], cu, 16, 4, 4, 4)
    with pytest.raises(AssertionError, match="cu_seqlens_q"):
        lib.gqa_chunk(q[:1], pool, pool, pt, None, cu[:1], 1, 0.1, torch.empty_like(q[:1]))
    with pytest.raises(TypeError, match="k must be a tensor"):
        lib.gqa_prompt(q, None, k, cu, 0.1, torch.empty_like(q))
    with pytest.raises(AssertionError, match=r"\[T, Hkv, D\]"):
        lib.gqa_prompt(q, pool, pool, cu, 0.1, torch.empty_like(q))
    with pytest.raises(AssertionError, match="heads that divide"):
        lib.gqa_prompt(q, torch.zeros((4, 3, 64), dtype=torch.bfloat16), torch.zeros((4, 3, 64), dtype=torch.bfloat16), cu, 0.1, torch.empty_like(q))


def test_step_refuses_shared_rows_and_missing_pages():
    table = PagedTokenTable(4, 16, torch.zeros((3, 64), dtype=torch.int32))
    with pytest.raises(AssertionError, match="rows of their own"):
        table.allocate_step([Req(table_idx=1, cached_len=0, device_len=1), Req(table_idx=1, cached_len=0, device_len=1)])
    with pytest.raises(RuntimeError, match="out of KV pages: 5 needed, 4 free"):
        table.allocate_step([Req(table_idx=0, cached_len=0, device_len=17), Req(table_idx=1, cached_len=0, device_len=33)])
    with pytest.raises(AssertionError, match="has requests"):
        table.allocate_step([])
    with pytest.raises(AssertionError, match="holds 64 tokens"):
        table.allocate_step([Req(table_idx=0, cached_len=65, device_len=66)])
    assert table.free_pages == 4


def test_oracle_attention_against_torch():
    gen = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn((n, h, 64), generator=gen, dtype=torch.float64) for n, h in ((5, 6), (12, 2), (12, 2)))
    ref = R.attend(q, k, v, 0.3)
    mask = torch.arange(12) <= 7 + torch.arange(5)[:, None]
    wide = lambda x: x.repeat_interleave(3, 1).transpose(0, 1)  # noqa: E731
    want = torch.nn.functional.scaled_dot_product_attention(q.transpose(0, 1), wide(k), wide(v), attn_mask=mask, scale=0.3)
    torch.testing.assert_close(ref.out, want.transpose(0, 1))
    s = torch.einsum("ihd,hjd->hij", q, wide(k)) * 0.3
    torch.testing.assert_close(ref.lse, torch.logsumexp(s.masked_fill(~mask, -float("inf")), -1).t())
    none = R.attend(q, k[:3], v[:3], 0.3)
    assert (none.out[:2] == 0).all() and none.lse[:2].isinf().all() and none.lse[2:].isfinite().all()


def test_oracle_tables_against_the_allocator():
    table = torch.zeros((4, 64), dtype=torch.int32)
    host = PagedTokenTable(12, 8, table.clone())
    free = host.free_slots.clone()
    reqs = [Req(table_idx=2, cached_len=0, device_len=19), Req(table_idx=0, cached_len=0, device_len=8)]
    host.allocate_paged(reqs)
    ref = R.step_tables(table, [2, 0], [0, 0], [19, 8], free, 8, 3, 2)
    assert torch.equal(ref.token_table, host.page_table) and ref.out_loc == host.out_loc(reqs).tolist()
    assert ref.pages_taken == 4 and ref.page_table.tolist() == [[0, 1, 2], [3, 0, 0]]


def test_launches_past_2_to_32_threads_are_refused_before_the_first():
    """The joining of split keys, a launch of its own, holds more threads here than the attention's; it was refused when
    that was launched already."""
    wide = dict(qt=2016 * 128, kr=63 * 128, vr=63 * 128, hq=2016, hk=63, ot=2016 * 128, lt=2016, cols=400, pts=400)
    for rc in (decode(batch=65535, **wide), chunk(batch=65535, T=65535, max_q=1, **wide)):
        assert rc == UNSUPPORTED and "more than a launch holds" in lib.load_library().mla_last_error().decode()
    rc = prompt(T=1 << 19, hq=4096, hk=4096, qt=4096 * 128, kr=4096 * 128, vr=4096 * 128, ot=4096 * 128, lt=4096)
    assert rc == UNSUPPORTED and "total_q * q_heads" in lib.load_library().mla_last_error().decode()
    rc = prompt(T=(1 << 19) - 1, batch=65535, hq=4096, hk=4096, qt=4096 * 128, kr=4096 * 128, vr=4096 * 128, ot=4096 * 128, lt=4096)
    assert rc == UNSUPPORTED and "more than a launch holds" in lib.load_library().mla_last_error().decode()


def test_step_refuses_rows_that_are_not_there_and_rows_of_the_padding():
    """The launch cuts a row index to the table, so that one past it would be another request's row; a row that is filled
    while padding reads it would be read half filled."""
    table = PagedTokenTable(4, 16, torch.zeros((3, 64), dtype=torch.int32))
    one = Req(table_idx=1, cached_len=0, device_len=1)
    for idx in (3, -1):
        far = Req(table_idx=idx, cached_len=0, device_len=1)
        for reqs, padding in (([one, far], []), ([one], [far])):
            with pytest.raises(AssertionError, match="has 3 rows"):
                table.allocate_step(reqs, padding)
    with pytest.raises(AssertionError, match="rows of their own"):
        table.allocate_step([one], [Req(table_idx=2, cached_len=0, device_len=1), Req(table_idx=1, cached_len=0, device_len=1)])
    assert table.free_pages == 4
