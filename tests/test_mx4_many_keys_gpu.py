"""Very long requests over the 4-bit cache: values of the largest size, whose sums pass fp32's range on the way unless the numerators
leave room for as many keys as a wave takes. The page table repeats two pages, keys of a lower and of a higher score."""

from __future__ import annotations

import math

import pytest
import torch

from minisgl_amd.kernel import lib
from test_mx4_gpu import DEV, i32

pytestmark = pytest.mark.gpu
HEADS, DIM, PS = 16, 64, 32
SCALE = 0.6931471824645996  # times log2(e), rounded, 1: scores are q . k in the log2 domain


def run(length, low, high):
    """Scores of the pages' keys: codes and scales of dims 0 and 32, as (code, scale, code, scale). Three tiles in 64 have the
    lower score, at random: so do the first tiles of some waves, to which numerators are relative then."""
    assert (torch.tensor(SCALE) * torch.tensor(math.log2(math.e), dtype=torch.float32)).item() == 1.0
    k, v = (lib.mx4_pool(2, PS, HEADS, DIM, DEV) for _ in "kv")
    k.codes.zero_(), v.codes.fill_(0x77), v.scales.fill_(252)  # 6 2^125
    for page, (c0, s0, c1, s1) in enumerate((low, high)):
        k.codes[page, :, :, 0], k.codes[page, :, :, 16] = c0, c1
        k.scales[page, :, :, 0], k.scales[page, :, :, 1] = s0, s1
    q = torch.zeros((1, HEADS, DIM), dtype=torch.bfloat16, device=DEV)
    q[..., 0] = q[..., 32] = 1.0
    gen = torch.Generator(device=DEV).manual_seed(0)
    pt = (torch.rand((1, length // PS), generator=gen, device=DEV) > 3 / 64).int()
    out, lse = torch.empty_like(q), torch.empty((1, HEADS), device=DEV)
    lib.gqa_decode_mx4(q, k, v, pt, i32([length]), SCALE, out, lse)
    return out.double().cpu(), lse.double().cpu(), PS * pt.sum().item()


@pytest.mark.parametrize("length", [1 << 16, 1 << 24])
def test_scores_whose_spacing_is_more_than_the_lag(length):
    """Scores of 1.5 2^26 and 8 more, fp32's spacing there: the higher ones are 2^8 times the lower, and references follow them.
    2^17 keys a wave (it has a 128th of them), of 2^-24 each where they do: half of what fp32 holds of this size."""
    out, lse, n = run(length, (7, 127 + 24, 0, 127), (7, 127 + 24, 6, 128))
    want = 6 * 2.0 ** 125
    # numerators are powers of two, sums over keys a rounding of 2^-23 (or a bit cut) for each of a wave's tiles, and the result's half step
    bound = (length / 128 / 32 + 16) * 2.0 ** -23 + 2.0 ** -8
    assert ((out - want).abs() <= bound * want).all()
    assert ((lse - (1.5 * 2 ** 26 + 8) * math.log(2) - math.log(n)).abs() <= 16).all()  # two steps of fp32 there


@pytest.mark.parametrize("length", [1 << 16, 3 << 25])
def test_more_keys_than_fit_a_fixed_room(length):
    """Scores of 0 and 6: the higher ones are at the lag's end, numerators 2^6, and up to 786,432 of them a wave."""
    out, lse, n = run(length, (0, 127, 0, 127), (0, 127, 7, 127))
    want = 6 * 2.0 ** 125
    bound = (length / 128 / 32 + 16) * 2.0 ** -23 + 2.0 ** -8
    assert ((out - want).abs() <= bound * want).all()
    assert ((lse - math.log(64.0 * n + (length - n))).abs() <= bound + 2.0 ** -18).all()
