"""Norms, rotation and cache rows of grouped heads on the GPU against the 64-bit oracle, within the bounds derived there."""

from __future__ import annotations

import pytest
import torch

from minisgl_amd.kernel import lib
from oracle import ref_mx4 as M

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
NAN = float("nan")
EPS = 1e-6


def randn(gen, *shape):
    return torch.randn(shape, generator=gen).to(torch.bfloat16)


def table(rotary, positions=300):
    angle = torch.arange(positions)[:, None] * 0.01 ** (torch.arange(rotary // 2) / max(rotary // 2, 1))
    return torch.cat((angle.cos(), angle.sin()), 1).float().contiguous()


def near(got, want, bound):
    over = (got.cpu().double() - want).abs() - bound
    assert over.max() <= 0, f"{over.max():.3e} past its bound"


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads", [(1, 1), (3, 1), (8, 2), (14, 2), (28, 4), (64, 8)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("normed", [False, True])
def test_heads(dim, heads, interleaved, normed):
    gen = torch.Generator().manual_seed(heads[0] + dim)
    hq, hk = heads
    for T, rotary in ((1, dim), (5, dim // 2), (67, dim), (3, 8)):
        qkv = randn(gen, T, (hq + 2 * hk) * dim)
        q, k, v = (x.unflatten(1, (-1, dim)) for x in qkv.to(DEV).split([hq * dim, hk * dim, hk * dim], 1))
        qw, kw = (randn(gen, dim), randn(gen, dim)) if normed else (None, None)
        pos, cs = torch.randint(0, 300, (T,), generator=gen, dtype=torch.int32), table(rotary)
        ps = 4
        pages = T // ps + 2
        slots = torch.randperm(pages * ps, generator=gen)[:T]
        pools = [torch.full((pages, ps, hk, dim), NAN, dtype=torch.bfloat16, device=DEV) for _ in "kv"]
        q_out = torch.full((T, hq, dim), NAN, dtype=torch.bfloat16, device=DEV)
        dev = lambda x: None if x is None else x.to(DEV)  # noqa: E731
        lib.qk_norm_rope(q, k, v, dev(qw), dev(kw), EPS, pos.to(DEV), cs.to(DEV), interleaved, q_out, *pools, slots=slots.to(DEV))
        raw_q, raw_k, raw_v = (x.unflatten(1, (-1, dim)) for x in qkv.split([hq * dim, hk * dim, hk * dim], 1))
        near(q_out, *M.norm_rope(raw_q, qw, EPS, pos, cs, interleaved))
        flat = [x.flatten(0, 1).cpu() for x in pools]
        near(flat[0][slots], *M.norm_rope(raw_k, kw, EPS, pos, cs, interleaved))
        assert torch.equal(flat[1][slots], raw_v)
        rest = torch.ones(pages * ps, dtype=torch.bool)
        rest[slots] = False
        assert all(x[rest].isnan().all() for x in flat)
        assert torch.equal(qkv.view(torch.int16), torch.cat([x.flatten(1) for x in (q, k, v)], 1).cpu().view(torch.int16))


@pytest.mark.parametrize("dim,rotary,interleaved", [(128, 128, False), (128, 64, True), (64, 64, False), (64, 16, False)])
def test_in_place(dim, rotary, interleaved):
    """q_out = q and k_out = k, parts of one projection's output; v without v_out stays, and no rotation at all is a copy."""
    gen = torch.Generator().manual_seed(dim)
    T, hq, hk = 333, 6, 2
    qkv = randn(gen, T, (hq + 2 * hk) * dim)
    q, k, v = (x.unflatten(1, (-1, dim)) for x in qkv.to(DEV).split([hq * dim, hk * dim, hk * dim], 1))
    raw_q, raw_k, raw_v = (x.unflatten(1, (-1, dim)) for x in qkv.split([hq * dim, hk * dim, hk * dim], 1))
    qw, kw, pos, cs = randn(gen, dim), randn(gen, dim), torch.randint(0, 300, (T,), generator=gen, dtype=torch.int32), table(rotary)
    lib.qk_norm_rope(q, k, None, qw.to(DEV), kw.to(DEV), EPS, pos.to(DEV), cs.to(DEV), interleaved, q, k)
    near(q, *M.norm_rope(raw_q, qw, EPS, pos, cs, interleaved))
    near(k, *M.norm_rope(raw_k, kw, EPS, pos, cs, interleaved))
    assert torch.equal(v.cpu(), raw_v)
    out = [torch.empty_like(x) for x in (q, k, v)]
    lib.qk_norm_rope(q, k, v, None, None, EPS, pos.to(DEV), table(0).to(DEV), interleaved, *out)
    assert all(torch.equal(a, b) for a, b in zip(out, (q, k, v)))


def test_slots_and_positions_outside():
    """Slots outside the pool are skipped, as a padded step's -1; positions are clamped into the table."""
    gen = torch.Generator().manual_seed(5)
    T, hq, hk, dim = 6, 4, 2, 128
    q, k, v = randn(gen, T, hq, dim), randn(gen, T, hk, dim), randn(gen, T, hk, dim)
    pos = torch.tensor([0, -5, 299, 300, 1 << 30, 7], dtype=torch.int32)
    cs, w = table(dim), randn(gen, dim)
    for dtype in (torch.int32, torch.int64):
        slots = torch.tensor([3, -1, 0, 8, 7, 2], dtype=dtype)
        pools = [torch.full((2, 4, hk, dim), NAN, dtype=torch.bfloat16, device=DEV) for _ in "kv"]
        q_out = torch.empty_like(q, device=DEV)
        lib.qk_norm_rope(q.to(DEV), k.to(DEV), v.to(DEV), w.to(DEV), w.to(DEV), EPS, pos.to(DEV), cs.to(DEV), False, q_out, *pools, slots=slots.to(DEV))
        want, bound = M.norm_rope(k, w, EPS, pos, cs, False)
        near(q_out, *M.norm_rope(q, w, EPS, pos, cs, False))
        stored = {3: 0, 0: 2, 7: 4, 2: 5}
        for row in range(8):
            got = [x.view(8, hk, dim)[row].cpu() for x in pools]
            if row in stored:
                near(got[0], want[stored[row]], bound[stored[row]])
                assert torch.equal(got[1], v[stored[row]])
            else:
                assert got[0].isnan().all() and got[1].isnan().all()


def test_strided_pools_and_no_tokens():
    """Pools with room between rows and heads, keys alone, and a call without tokens."""
    gen = torch.Generator().manual_seed(6)
    T, hq, hk, dim = 9, 5, 3, 64
    q, k = randn(gen, T, hq, dim), randn(gen, T, hk, dim)
    big = torch.full((5, 4, hk, dim + 16), NAN, dtype=torch.bfloat16, device=DEV)
    pos, cs, w = torch.arange(T, dtype=torch.int32), table(dim), randn(gen, dim)
    slots = torch.randperm(20, generator=gen)[:T]
    q_out = torch.full((hq, T, dim), NAN, dtype=torch.bfloat16, device=DEV)
    args = (w.to(DEV), w.to(DEV), EPS, pos.to(DEV), cs.to(DEV), True, q_out.transpose(0, 1), big[..., :dim])
    lib.qk_norm_rope(q.to(DEV), k.to(DEV), None, *args, slots=slots.to(DEV))
    near(q_out.transpose(0, 1), *M.norm_rope(q, w, EPS, pos, cs, True))
    near(big.view(20, hk, -1)[slots.to(DEV), :, :dim], *M.norm_rope(k, w, EPS, pos, cs, True))
    assert big[..., dim:].isnan().all()
    none = torch.empty((0, hq, dim), dtype=torch.bfloat16, device=DEV)
    lib.qk_norm_rope(none, none[:, :hk], None, None, None, EPS, pos[:0].to(DEV), cs.to(DEV), False, none, none[:, :hk])


def test_special_values():
    """NaN and infinities stay in their head; a row of zeros is 0; small and large rows."""
    gen = torch.Generator().manual_seed(7)
    dim, w = 128, torch.ones(128, dtype=torch.bfloat16)
    q = randn(gen, 8, 4, dim)
    q[1, 2, 5], q[2, 0, 127], q[3, 1] = NAN, float("inf"), 0.0
    q[4] *= 1e15
    q[5] *= 1e-12
    pos, cs = torch.zeros(8, dtype=torch.int32), table(dim)
    out = torch.empty_like(q, device=DEV)
    k_out = torch.empty_like(q[:, :1], device=DEV)
    lib.qk_norm_rope(q.to(DEV), q[:, :1].to(DEV), None, w.to(DEV), w.to(DEV), EPS, pos.to(DEV), cs.to(DEV), False, out, k_out)
    hit = torch.zeros((8, 4), dtype=torch.bool)
    hit[1, 2] = hit[2, 0] = True
    got = out.cpu()
    assert got[1, 2].isnan().all() and got[2, 0, 127].isnan() and (got[3, 1] == 0).all()
    want, bound = M.norm_rope(q, w, EPS, pos, cs, False)
    near(got[~hit], want[~hit], bound[~hit])


def test_captured():
    gen = torch.Generator().manual_seed(8)
    T, hq, hk, dim = 40, 8, 2, 128
    qkv = torch.empty((T, (hq + 2 * hk) * dim), dtype=torch.bfloat16, device=DEV)
    q, k, v = (x.unflatten(1, (-1, dim)) for x in qkv.split([hq * dim, hk * dim, hk * dim], 1))
    w, cs = randn(gen, dim), table(dim)
    pos, slots = torch.zeros(T, dtype=torch.int32, device=DEV), torch.zeros(T, dtype=torch.int32, device=DEV)
    pools = [torch.zeros((20, 4, hk, dim), dtype=torch.bfloat16, device=DEV) for _ in "kv"]
    q_out, wd, cd = torch.empty((T, hq, dim), dtype=torch.bfloat16, device=DEV), w.to(DEV), cs.to(DEV)
    call = lambda: lib.qk_norm_rope(q, k, v, wd, wd, EPS, pos, cd, False, q_out, *pools, slots=slots)  # noqa: E731
    graph = torch.cuda.CUDAGraph()
    slots.copy_(torch.arange(T))
    call()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        call()
    for _ in range(3):
        raw = randn(gen, T, (hq + 2 * hk) * dim)
        p, s = torch.randint(0, 300, (T,), generator=gen, dtype=torch.int32), torch.randperm(80, generator=gen)[:T].int()
        qkv.copy_(raw), pos.copy_(p), slots.copy_(s)
        graph.replay()
        torch.cuda.synchronize()
        raw_q, raw_k, raw_v = (x.unflatten(1, (-1, dim)) for x in raw.split([hq * dim, hk * dim, hk * dim], 1))
        near(q_out, *M.norm_rope(raw_q, w, EPS, p, cs, False))
        near(pools[0].view(80, hk, dim)[s.to(DEV).long()], *M.norm_rope(raw_k, w, EPS, p, cs, False))
        assert torch.equal(pools[1].view(80, hk, dim)[s.to(DEV).long()].cpu(), raw_v)


def test_another_stream():
    gen = torch.Generator().manual_seed(9)
    T, hq, hk, dim = 700, 4, 2, 128
    q, k, w = randn(gen, T, hq, dim), randn(gen, T, hk, dim), randn(gen, dim)
    pos, cs = torch.arange(T, dtype=torch.int32) % 300, table(dim)
    qd, kd, wd, pd, cd = q.to(DEV), k.to(DEV), w.to(DEV), pos.to(DEV), cs.to(DEV)
    late, q_out, k_out, side = torch.zeros_like(qd), torch.zeros_like(qd), torch.zeros_like(kd), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(1_000_000)
        late.copy_(qd)
    lib.qk_norm_rope(late, kd, None, wd, wd, EPS, pd, cd, False, q_out, k_out, stream=side)
    side.synchronize()
    near(q_out, *M.norm_rope(q, w, EPS, pos, cs, False))
    near(k_out, *M.norm_rope(k, w, EPS, pos, cs, False))


def test_tensors_that_do_not_fit():
    x, k, w = (torch.zeros(s, dtype=torch.bfloat16, device=DEV) for s in ((3, 4, 128), (3, 2, 128), (128,)))
    i, cs = torch.zeros(3, dtype=torch.int32, device=DEV), table(128).to(DEV)
    pool = torch.zeros((2, 4, 2, 128), dtype=torch.bfloat16, device=DEV)
    call = lambda q=x, k=k, v=None, qw=w, kw=w, pos=i, cs=cs, q_out=x, k_out=k, v_out=None, **kv: lib.qk_norm_rope(  # noqa: E731
        q, k, v, qw, kw, EPS, pos, cs, False, q_out, k_out, v_out, **kv)
    for kw, text in ((dict(v=k), "v comes with"), (dict(qw=None), "both weights"), (dict(qw=w[:64]), "weights"), (dict(pos=i.long()), "positions"),
                     (dict(cs=cs.double()), "cos_sin"), (dict(cs=cs[:, :64]), "cos_sin"), (dict(q_out=k), "q_out"), (dict(k_out=x), "k_out"), (dict(k=k[:2]), "k must"),
                     (dict(k_out=pool), "k_out"), (dict(slots=i), "pools"), (dict(slots=i.float(), k_out=pool), "slots"), (dict(q=x.float()), "q must"),
                     (dict(slots=i, k_out=pool, v=k, v_out=pool[:1]), "as many rows")):
        with pytest.raises(AssertionError, match=text):
            call(**kw)
    with pytest.raises(lib.MLAKernelError, match="overlap"):
        call(q_out=x[:1].expand(3, 4, 128))
    with pytest.raises(lib.MLAKernelError, match="rotary_dim"):
        call(cs=cs[:, :12].contiguous())


def test_factors_past_the_range():
    """1 / norm times the weight may leave fp32's range where the result does not."""
    gen = torch.Generator().manual_seed(10)
    T, hq, hk, dim = 9, 3, 1, 128
    pos, cs = torch.arange(T, dtype=torch.int32), table(dim)
    for x, w in ((1e18, 1e-30), (1e-9, 3e36)):
        q, k = randn(gen, T, hq, dim) * x, randn(gen, T, hk, dim) * x
        qw, kw = randn(gen, dim) * w, randn(gen, dim) * w
        q_out, k_out = (torch.full(z.shape, NAN, dtype=torch.bfloat16, device=DEV) for z in (q, k))
        lib.qk_norm_rope(q.to(DEV), k.to(DEV), None, qw.to(DEV), kw.to(DEV), EPS, pos.to(DEV), cs.to(DEV), False, q_out, k_out)
        near(q_out, *M.norm_rope(q, qw, EPS, pos, cs, False))
        near(k_out, *M.norm_rope(k, kw, EPS, pos, cs, False))
