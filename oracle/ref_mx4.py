"""64-bit oracle of the 4-bit cache and of the norms and rotation of grouped heads. TEST INFRASTRUCTURE ONLY.

4 bits: MXFP4 of the OCP Microscaling Formats 1.0, by its tables: E2M1 elements, E8M0 scales, blocks of 32.
Norms and rotation: python/minisgl/layers/attention.py:17-57, norm.py and rotary.py:22-51 of the reference.
"""

from __future__ import annotations

import torch

# of codes 0 to 15: E2M1 has one bit of mantissa and an exponent's bias of 1
ELEMENTS = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64)


def rounded(x: torch.Tensor):
    """Codes ``[..., D / 2]`` and scales ``[..., D / 32]`` (uint8) of bf16 rows ``x [..., D]``, a value at a time by its
    distance to every code."""
    b = x.double().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1)
    bad = ~torch.isfinite(b).all(-1)
    # floor(log2 top): frexp gives top = m 2^e with m in [1/2, 1)
    e = torch.where(top > 0, torch.frexp(torch.where(bad, 1.0, top)).exponent - 1, -1000) - 2
    e = torch.where(bad, 0, e.clamp_min(-127))
    y = torch.where(bad[..., None], 0.0, b) * 2.0 ** (-e.double())[..., None]
    far = (y.abs()[..., None] - ELEMENTS[:8]).abs()
    near = far.amin(-1, keepdim=True)
    tied = far == near  # two neighbours at most, one of them even
    even = torch.arange(8) % 2 == 0
    code = torch.where((tied & even).any(-1), (tied & even).int().argmax(-1), tied.int().argmax(-1))
    code = torch.where(torch.signbit(y) & ~bad[..., None], code + 8, code).flatten(-2)
    scales = torch.where(bad, 255, e + 127)
    return (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8), scales.to(torch.uint8)


def values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """float64 ``[..., D]``."""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
    unit = torch.where(scales == 255, float("nan"), 2.0 ** (scales.double() - 127))
    return (ELEMENTS[c].unflatten(-1, (-1, 32)) * unit[..., None]).flatten(-2)


def norm_rope(x, weight, eps: float, positions, cos_sin, interleaved: bool):
    """``x [T, H, D]`` normed (``weight`` None: not) and rotated, and how far a bf16 result of fp32 arithmetic may be from it.

    The sum of D squares, the root and three products are off by at most (D + 8) 2^-24 of the value together; a rotation adds
    3 roundings of each of its two products' sizes; the last rounding is half a step of bf16, 2^-8 of the result. Values below
    bf16's normal range (2^-126) are off by half its smallest step, 2^-134."""
    y = x.double()
    D, R = x.shape[-1], cos_sin.shape[1]
    if weight is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * weight.double()
    at = cos_sin.double()[positions.long().clamp(0, cos_sin.shape[0] - 1)][:, None]
    c, s = at[..., : R // 2], at[..., R // 2 :]
    first, second = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, R // 2), slice(R // 2, R))
    a, b = y[..., first].clone(), y[..., second].clone()
    size = y.abs().clone()
    y = y.clone()
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    size[..., first], size[..., second] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    return y, 2.0 ** -8 * y.abs() + 1.01 * (D + 12) * 2.0 ** -24 * size + 2.0 ** -134
