"""Requests in pieces: the joining of their partial results, on the GPU."""

from __future__ import annotations

import pytest
import torch

from minisgl_amd.kernel import lib

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("size", [2.0 ** 126, 1.0])
def test_pieces_of_the_largest_values(dim, size):
    """Pieces of alike weights and values next to fp32's largest: their mean is inside it, their sum is not."""
    L, ps = 20000, 64
    pages = -(-L // ps)
    k = torch.zeros((pages, ps, 2, dim), dtype=torch.bfloat16, device=DEV)
    v = torch.full_like(k, size)
    q = torch.ones((1, 4, dim), dtype=torch.bfloat16, device=DEV)
    out, lse = torch.empty_like(q), torch.empty((1, 4), device=DEV)
    pt = torch.arange(pages, dtype=torch.int32, device=DEV)[None]
    lib.gqa_decode(q, k, v, pt, torch.tensor([L], dtype=torch.int32, device=DEV), 0.1, out, lse)
    assert (out.double() == size).all()  # numerators are 1, and the mean is exact but for roundings far below bf16's
    want = torch.log(torch.tensor(float(L), dtype=torch.float64))
    # every sum is of whole numbers below 2^24: two logarithms and a product, half a step and an ulp of fp32 each
    assert ((lse.double().cpu() - want).abs() <= 2.0 ** -21 * want).all()
