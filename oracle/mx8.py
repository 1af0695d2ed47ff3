"""The 8-bit form of activations and weights in float64: e4m3 values, every 32 of a row under one power-of-two scale.

Pinned by torch's own cast to float8_e4m3fn and by the definition of the scale (``tests/test_mx8_refusals.py``).
"""
from __future__ import annotations

import torch

BLOCK = 32


def power(e: torch.Tensor) -> torch.Tensor:
    """2^e in float64, exactly (e a whole number in -1022 .. 1023)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def scale_exponents(v: torch.Tensor) -> torch.Tensor:
    """[rows, cols] float64 -> int64 [rows, cols / 32]: the smallest e >= -127 with largest |v| / 2^e <= 448."""
    largest = v.view(v.size(0), v.size(1) // BLOCK, BLOCK).abs().amax(-1)
    part, e = torch.frexp(largest)              # 448 is 7/8 of 2^9
    return torch.where(largest == 0, -127, (e.long() - 9 + (part > 0.875)).clamp(min=-127))


def quantize(v: torch.Tensor):
    """Values that the 8-bit form of v [rows, cols] (float64) stands for, and its exponents.  A block with an infinity or a NaN is NaN."""
    b = v.view(v.size(0), v.size(1) // BLOCK, BLOCK)
    bad = ~b.isfinite().all(-1)
    b = torch.where(bad[..., None], 0.0, b)
    e = scale_exponents(b.reshape(v.shape))
    s = power(e[..., None])
    r = b / s
    step = power((torch.frexp(r)[1] - 1).clamp(min=-6) - 3)
    q = torch.round(r / step) * step * s        # (torch rounds ties to even)
    return torch.where(bad[..., None], float("nan"), q).view(v.shape), torch.where(bad, 128, e)


def exponents_of(scales: torch.Tensor, cols: int) -> torch.Tensor:
    """The same exponents from the bytes [ceil(cols / 128), rows, 4] of the package (NaN: 128)."""
    return scales.permute(1, 0, 2).reshape(scales.size(1), 4 * scales.size(0))[:, :cols // BLOCK].long() - 127


def silu(g):
    return g * torch.sigmoid(g)


def swiglu_gradient(gate, up, dh):
    s = torch.sigmoid(gate)
    return torch.cat((dh * up * s * (1 + gate * (1 - s)), dh * gate * s), -1)


def norm_gradient(h, gamma, dy, dh, eps):
    """Gradients of h's RMSNorm: (d h with dh added, d gamma)."""
    rstd = (h.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
    n, g = h * rstd, dy * gamma
    return rstd * (g - n * (g * n).mean(-1, keepdim=True)) + dh, (dy * n).sum(0)
