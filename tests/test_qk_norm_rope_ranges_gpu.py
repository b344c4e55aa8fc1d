"""Norms of rows whose squares leave fp32's range: every finite row has its norm, with any eps."""

from __future__ import annotations

import pytest
import torch

from minisgl_amd.kernel import lib
from oracle import ref_mx4 as M
from test_qk_norm_rope_gpu import DEV, NAN, near, randn, table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("eps", [0.0, 2.0 ** -140, 2.0 ** -110, 2.0 ** -99, 1e-6, 2.0 ** 127])
def test_rows_of_every_size(dim, interleaved, eps):
    """A row for each power of two, the largest and the smallest of bf16 among them, and rows of one value beside much smaller ones.
    The bounds are those of any row: a root of 2^-128 has 21 bits, 2^-21 = 8 2^-24 of the D + 12 that are allowed, of which a lane's
    8 squares, 4 sums over lanes and the products take 16."""
    gen = torch.Generator().manual_seed(dim)
    sizes = torch.cat((2.0 ** torch.arange(-131, 126).double(), 2.0 ** torch.arange(-131, 126).double()))
    T, hq, hk = len(sizes), 3, 1
    x = torch.randn((T, hq + hk, dim), generator=gen).double().clamp(-3.9, 3.9)
    x[T // 2 :, :, 1:] *= 2.0 ** -30  # one large value
    x[x == 0] = 0.5
    x = (x * sizes[:, None, None]).to(torch.bfloat16)
    x[5, 0], x[T // 2 - 1, 0] = torch.finfo(torch.bfloat16).max, -torch.finfo(torch.bfloat16).max
    x[6, 0], x[7, 0] = 2.0 ** -133, -(2.0 ** -133)
    x[:, :, 0] = torch.where(x[:, :, 0] == 0, torch.tensor(2.0 ** -133, dtype=torch.bfloat16), x[:, :, 0])  # no row of zeros
    q, k = x[:, :hq], x[:, hq:]
    qw, kw = randn(gen, dim), randn(gen, dim)
    pos, cs = torch.arange(T, dtype=torch.int32) % 300, table(dim)
    q_out, k_out = (torch.full(z.shape, NAN, dtype=torch.bfloat16, device=DEV) for z in (q, k))
    lib.qk_norm_rope(q.to(DEV), k.to(DEV), None, qw.to(DEV), kw.to(DEV), eps, pos.to(DEV), cs.to(DEV), interleaved, q_out, k_out)
    near(q_out, *M.norm_rope(q, qw, eps, pos, cs, interleaved))
    near(k_out, *M.norm_rope(k, kw, eps, pos, cs, interleaved))


def test_rows_of_zeros_infinities_and_nan():
    """Zeros with an eps are zeros; without, 0 / 0. An infinity or a NaN makes its head's dim NaN, and only that head."""
    gen = torch.Generator().manual_seed(3)
    dim = 128
    w, pos, cs = torch.ones(dim, dtype=torch.bfloat16, device=DEV), torch.zeros(6, dtype=torch.int32, device=DEV), table(dim).to(DEV)
    q = randn(gen, 6, 4, dim) * 1e30
    q[0, 1], q[1, 2, 7], q[2, 3, 9], q[3, 0] = 0.0, float("inf"), NAN, 1.0
    for eps in (0.0, 2.0 ** -120, 1e-6):
        out, k_out = torch.full_like(q, 5.0, device=DEV), torch.empty_like(q[:, :1], device=DEV)
        lib.qk_norm_rope(q.to(DEV), q[:, :1].to(DEV), None, w, w, eps, pos, cs, False, out, k_out)
        got = out.cpu()
        assert got[0, 1].isnan().all() if eps == 0 else (got[0, 1] == 0).all()
        assert got[1, 2, 7].isnan() and got[2, 3].isnan().all()
        rest = torch.ones((6, 4), dtype=torch.bool)
        rest[0, 1] = rest[1, 2] = rest[2, 3] = False
        want, bound = M.norm_rope(q, w.cpu(), eps, pos.cpu(), cs.cpu(), False)
        near(got[rest], want[rest], bound[rest])
