"""Refusals of the 4-bit cache's and the rotation's entry points, made on the host before anything is launched (the device
pointers here need not be any), the workspace's size, and the oracle's own checks."""

from __future__ import annotations

import ctypes

import pytest
import torch

from minisgl_amd.kernel import lib
from oracle import ref_mx4 as M

P = 1 << 20  # a 16-byte aligned address, never followed
OK, INVALID, UNSUPPORTED = 0, 1, 3


class Pool(ctypes.Structure):
    _fields_ = [("codes", ctypes.c_void_p), ("scales", ctypes.c_void_p)] + [(n, ctypes.c_int64) for n in ("cp", "ct", "ch", "sp", "st", "sh")]


def pool(**kw):
    a = dict(codes=P, scales=P, cp=16 * 128, ct=128, ch=64, sp=16 * 8, st=8, sh=4)
    assert set(kw) <= set(a)
    a.update(kw)
    return Pool(*a.values())


def rows(entry, kp=None, vp=None, **kw):
    a = dict(k_pool=ctypes.byref(kp or pool()), v_pool=ctypes.byref(vp or pool()), pages=10, ps=16, heads=2, d=128, idx=P, bits=32, n=5, k=P, kt=256, kh=128,
             v=P, vt=256, vh=128, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return getattr(lib.load_library(), entry)(*a.values())


def chunk(kp=None, vp=None, **kw):
    a = dict(q=P, qt=1024, qh=128, k_pool=ctypes.byref(kp or pool()), v_pool=ctypes.byref(vp or pool()), pages=10, ps=16, pt=P, cols=4, pts=4, cu=P, lens=P,
             batch=2, T=10, max_q=8, total=128, hq=8, hk=2, d=128, scale=0.1, ws=P, ws_bytes=1 << 40, out=P, ot=1024, oh=128, lse=P, lt=8, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.load_library().mla_gqa_chunk_mx4(*a.values())


def decode(kp=None, vp=None, **kw):
    a = dict(q=P, qt=1024, qh=128, k_pool=ctypes.byref(kp or pool()), v_pool=ctypes.byref(vp or pool()), pages=10, ps=16, pt=P, cols=4, pts=4, lens=P,
             batch=2, total=128, hq=8, hk=2, d=128, scale=0.1, ws=P, ws_bytes=1 << 40, out=P, ot=1024, oh=128, lse=P, lt=8, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.load_library().mla_gqa_decode_mx4(*a.values())


def rope(**kw):
    a = dict(q=P, qt=1024, qh=128, k=P, kt=256, kh=128, v=P, vt=256, vh=128, qw=P, kw=P, eps=1e-6, pos=P, cs=P, max_pos=100, rotary=128, inter=0, T=5, hq=8,
             hk=2, d=128, qo=P, qot=1024, qoh=128, ko=P, kor=256, koh=128, vo=P, vor=256, voh=128, slots=P, bits=32, rows=160, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.load_library().mla_qk_norm_rope_bf16(*a.values())


POOLS = [
    (dict(kp=pool(codes=None)), INVALID, "null"), (dict(vp=pool(scales=None)), INVALID, "null"), (dict(k_pool=None), INVALID, "null"),
    (dict(kp=pool(codes=P + 8)), INVALID, "aligned"), (dict(vp=pool(scales=P + 2)), INVALID, "aligned"),
    (dict(kp=pool(ct=72)), INVALID, "strides"), (dict(kp=pool(ch=-64)), INVALID, "strides"), (dict(vp=pool(sh=2)), INVALID, "strides"), (dict(vp=pool(st=-8)), INVALID, "strides"),
    (dict(ps=24), UNSUPPORTED, "page_size"), (dict(ps=0), UNSUPPORTED, "page_size"), (dict(pages=0), INVALID, "num_pages"),
    (dict(pages=1 << 20, ps=1 << 12), UNSUPPORTED, "2^31 rows"), (dict(d=96), UNSUPPORTED, "head_dim"), (dict(d=256), UNSUPPORTED, "head_dim"),
    (dict(kp=pool(ct=1 << 25)), UNSUPPORTED, "16 MiB"), (dict(vp=pool(st=1 << 25)), UNSUPPORTED, "16 MiB"),
    (dict(kp=pool(cp=0)), INVALID, "over one another"), (dict(kp=pool(st=0)), INVALID, "over one another"), (dict(vp=pool(ch=48)), INVALID, "over one another"),
]
ROWS = POOLS + [
    (dict(n=-1), INVALID, "rows"), (dict(bits=16), INVALID, "index_bits"), (dict(idx=None), INVALID, "null"), (dict(k=None), INVALID, "null"), (dict(v=None), INVALID, "null"),
    (dict(k=P + 8), INVALID, "aligned"), (dict(kt=260), INVALID, "multiples"), (dict(vh=-128), INVALID, "multiples"), (dict(heads=0), INVALID, "kv_heads"),
    (dict(n=1 << 28, heads=16), UNSUPPORTED, "launch"),
]
ATTENTION = POOLS + [
    (dict(hq=8, hk=3), INVALID, "no multiple"), (dict(hq=0), INVALID, "no multiple"), (dict(batch=-1), INVALID, "batch"), (dict(total=-1), INVALID, "total_keys"),
    (dict(q=None), INVALID, "null"), (dict(out=None), INVALID, "null"), (dict(pt=None), INVALID, "null"), (dict(lens=None), INVALID, "null"), (dict(ws=None), INVALID, "null"),
    (dict(q=P + 8), INVALID, "aligned"), (dict(out=P + 4), INVALID, "aligned"), (dict(qt=1028), INVALID, "q strides"), (dict(oh=124), INVALID, "out strides"),
    (dict(vp=pool(ct=256)), INVALID, "same strides"), (dict(kp=pool(sp=256)), INVALID, "same strides"),
    (dict(cols=0), INVALID, "pt_cols"), (dict(pts=3), INVALID, "pt_stride"), (dict(lt=7), INVALID, "lse_stride"), (dict(scale=0.0), INVALID, "scale"),
    (dict(scale=float("nan")), INVALID, "scale"), (dict(ws=P + 8), INVALID, "workspace"), (dict(ws_bytes=1000), INVALID, "workspace"), (dict(batch=70000), UNSUPPORTED, "65535"),
]
ROPE = [
    (dict(T=-1), INVALID, "tokens"), (dict(hq=5000), INVALID, "q_heads"), (dict(hk=-1), INVALID, "kv_heads"), (dict(d=96), UNSUPPORTED, "head_dim"),
    (dict(rotary=132), INVALID, "rotary_dim"), (dict(rotary=136), INVALID, "rotary_dim"), (dict(rotary=12), INVALID, "rotary_dim"), (dict(rotary=-8), INVALID, "rotary_dim"),
    (dict(max_pos=0), INVALID, "max_position"), (dict(qw=None), INVALID, "weights"), (dict(v=None), INVALID, "v_out"), (dict(vo=None), INVALID, "v_out"),
    (dict(eps=-1.0), INVALID, "eps"), (dict(eps=float("nan")), INVALID, "eps"), (dict(bits=8), INVALID, "index_bits"), (dict(slots=None, rows=4), INVALID, "rows"),
    (dict(q=None), INVALID, "null"), (dict(k=None), INVALID, "null"), (dict(qo=None), INVALID, "null"), (dict(ko=None), INVALID, "null"), (dict(pos=None), INVALID, "null"),
    (dict(cs=None), INVALID, "null"), (dict(q=P + 8), INVALID, "aligned"), (dict(cs=P + 4), INVALID, "aligned"), (dict(vo=P + 2), INVALID, "aligned"),
    (dict(qt=1028), INVALID, "strides"), (dict(kor=-256), INVALID, "strides"), (dict(T=1 << 30), UNSUPPORTED, "launch"), (dict(rows=-1), INVALID, "out_rows"),
]


LOAD = ROWS + [(dict(kt=0), INVALID, "overlap"), (dict(vt=128), INVALID, "overlap"), (dict(kh=0), INVALID, "overlap")]
ROPE += [(dict(qot=2048), INVALID, "in the place"), (dict(qo=16 * P, ko=16 * P), INVALID, "no slots"), (dict(qo=16 * P, vo=16 * P), INVALID, "no slots"),
         (dict(slots=None, rows=5, kor=512), INVALID, "in the place")]
ELSE = dict(qo=16 * P, ko=32 * P, vo=48 * P)
ROPE += [({**ELSE, **kw}, INVALID, "overlap") for kw in (dict(qot=0), dict(qoh=64), dict(kor=128), dict(voh=0))]


@pytest.mark.parametrize("call,cases", [
    (lambda **kw: rows("mla_mx4_store", **kw), ROWS), (lambda **kw: rows("mla_mx4_load", **kw), LOAD), (decode, ATTENTION),
    (chunk, ATTENTION + [(dict(cu=None), INVALID, "null"), (dict(max_q=-1), INVALID, "max_q"), (dict(T=-1), INVALID, "total_q")]), (rope, ROPE)])
def test_refusals(call, cases):
    for kw, code, text in cases:
        rc, message = call(**kw), lib.load_library().mla_last_error().decode()
        assert rc == code and text in message, (kw, rc, message)


def test_empty_calls_do_nothing():
    assert rows("mla_mx4_store", n=0, idx=None, k=None) == OK and rows("mla_mx4_load", n=0, v=None) == OK
    assert decode(batch=0, q=None) == OK and chunk(T=0, cu=None) == OK and chunk(max_q=0) == OK
    assert rope(T=0, q=None) == OK and rope(hq=0, hk=0) == OK


def test_workspace_bytes():
    """Partial results alone for up to 512 rows a request; past that the values of total_keys keys and a table, not more than the
    page table holds, and never less for more."""
    assert lib.gqa_mx4_workspace_bytes(16, 32, 1, 128, 100, 1 << 17, 1 << 24) == lib.gqa_workspace_bytes(16, 32, 1, 128)
    at = lib.gqa_mx4_workspace_bytes(65, 64, 8, 128, 4, 8192, 20000)
    split = lib.gqa_workspace_bytes(65, 64, 8, 128)
    assert split + 2 * 20000 * 8 * 128 * 2 <= at <= split + 4 * 4 * 128 + 2 * (20000 + 4 * 64) * 8 * 128 * 2
    assert lib.gqa_mx4_workspace_bytes(65, 64, 8, 128, 4, 8192, 1 << 40) == lib.gqa_mx4_workspace_bytes(65, 64, 8, 128, 4, 8192, 4 * 8192)
    assert at <= lib.gqa_mx4_workspace_bytes(66, 64, 8, 128, 4, 8192, 20000) and at <= lib.gqa_mx4_workspace_bytes(65, 64, 8, 128, 5, 8192, 20001)
    assert lib.gqa_mx4_workspace_bytes(1 << 20, 4096, 4096, 128, 65535, 1 << 31, 1 << 62) > 0  # no overflow
    for bad in ((1, 8, 2, 128, 70000, 1, 1), (-1, 8, 2, 128, 1, 1, 1), (1, 8, 3, 128, 1, 1, 1), (1, 8, 2, 96, 1, 1, 1), (1, 8, 2, 128, -1, 1, 1), (1, 8, 2, 128, 1, -1, 1), (1, 8, 2, 128, 1, 1, -1)):
        with pytest.raises(lib.MLAKernelError):
            lib.gqa_mx4_workspace_bytes(*bad)


def test_tensors_that_do_not_fit():
    """On the host's side of the Python calls: tensors that are not on a GPU, before any entry point."""
    x = torch.zeros((2, 4, 128), dtype=torch.bfloat16)
    p = lib.mx4_pool(2, 4, 4, 128, "cpu")
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(AssertionError, match="GPU"):
        lib.mx4_store(p, p, i, x, x)
    with pytest.raises(AssertionError, match="GPU"):
        lib.mx4_load(p, p, i)
    with pytest.raises(AssertionError, match="GPU"):
        lib.gqa_decode_mx4(x, p, p, i.view(2, 1), i, 0.1, x)
    with pytest.raises(AssertionError, match="GPU"):
        lib.qk_norm_rope(x, x, None, None, None, 1e-6, i, torch.zeros((8, 128)), False, x, x)
    with pytest.raises(AssertionError, match="head_dim"):
        lib.mx4_pool(2, 4, 4, 96, "cpu")
    with pytest.raises(TypeError):
        lib.mx4_store(p, p, None, x, x)


def test_pool_layout():
    p = lib.mx4_pool(3, 16, 4, 128, "cpu")
    assert p.codes.shape == (3, 16, 4, 64) and p.scales.shape == (3, 16, 4, 4)
    assert p.codes.stride() == (16 * 4 * 64, 64, 16 * 64, 1) and p.scales.stride() == (16 * 4 * 4, 4, 16 * 4, 1)


def test_oracle_rounds_to_the_nearest():
    gen = torch.Generator().manual_seed(0)
    x = torch.randn((50, 128), generator=gen).to(torch.bfloat16)
    y = M.values(*M.rounded(x))
    top = x.double().view(50, 4, 32).abs().amax(-1, keepdim=True)
    unit = 2.0 ** (torch.floor(torch.log2(top)) - 2)
    off = (y - x.double()).view(50, 4, 32).abs() / unit
    size = x.double().view(50, 4, 32).abs() / unit
    # half a step: of 1/2 below 2 units, 1 below 4, 2 above; what passes 6 is cut
    half = torch.where(size < 2, 0.25, torch.where(size < 4, 0.5, 1.0))
    assert (off <= torch.where(size > 6, size - 6, half)).all() and off.max() < 2


@pytest.mark.parametrize("value,code", [(0.25, 0), (0.75, 2), (1.25, 2), (1.75, 4), (2.5, 4), (3.5, 6), (5.0, 6), (6.0, 7), (7.96875, 7), (0.265625, 1), (4.96875, 6), (5.03125, 7)])
def test_oracle_ties(value, code):
    x = torch.zeros(32)
    x[0], x[1], x[2] = 4.0, value, -value
    codes, scales = M.rounded(x.to(torch.bfloat16))
    assert scales.item() == 127 and codes[0] == 6 + 16 * code and codes[1] % 16 == (8 + code if value else 0)


def test_oracle_special_blocks():
    x = torch.zeros((4, 32))
    x[1, 3], x[2, 4], x[3] = float("nan"), float("inf"), 2.0 ** -133
    codes, scales = M.rounded(x.to(torch.bfloat16))
    assert scales.flatten().tolist() == [0, 255, 255, 0]
    assert M.values(codes, scales)[1:3].isnan().all() and (M.values(codes, scales)[3] == 0).all()


def test_oracle_rotation():
    """Two positions' dot product depends on their distance alone, and lengths are kept."""
    gen = torch.Generator().manual_seed(1)
    angle = torch.arange(64)[:, None] * 0.1 ** (torch.arange(32) / 32)
    cs = torch.cat((angle.cos(), angle.sin()), 1).float()
    x = torch.randn((1, 2, 64), generator=gen).to(torch.bfloat16)
    for inter in (False, True):
        at = [M.norm_rope(x, None, 0.0, torch.tensor([p]), cs, inter)[0] for p in (3, 10, 20, 27)]
        dots = [(at[i][0, 0] * at[j][0, 1]).sum() for i, j in ((0, 1), (2, 3))]
        torch.testing.assert_close(dots[0], dots[1], rtol=1e-5, atol=1e-5)
        torch.testing.assert_close(at[0].norm(), x.double().norm(), rtol=1e-6, atol=0)
    w = torch.full((64,), 2.0, dtype=torch.bfloat16)
    y, _ = M.norm_rope(x, w, 0.0, torch.tensor([5]), cs, False)
    torch.testing.assert_close(y.pow(2).mean(-1), torch.full((1, 2), 4.0, dtype=torch.float64), rtol=1e-6, atol=0)
