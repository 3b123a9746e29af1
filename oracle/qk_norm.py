"""Norms of q and k head by head with the rotation, in 64 bits, and how far a kernel may be off.

A row x of ``head_dim`` elements becomes y = x / sqrt(mean(x^2) + eps) * weight, and its first
``rotary_dim`` elements turn in pairs as :mod:`oracle.rope` says, by angles in 64 bits.
"""

from __future__ import annotations

import math

import torch


def frequencies(rotary_dim: int, rope_scale: float, rope_theta: float, llama31: dict | None) -> torch.Tensor:
    g = rope_theta ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    if not llama31:
        return g / rope_scale
    lo, hi = float(llama31["low_freq_factor"]), float(llama31["high_freq_factor"])
    smooth = ((float(llama31["old_context_len"]) * g / (2 * math.pi) - lo) / (hi - lo)).clamp(0, 1)
    return (1 - smooth) * g / rope_scale + smooth * g


def norm_rope(x: torch.Tensor, weight: torch.Tensor, pos: torch.Tensor, eps: float, rotary_dim: int, interleave: bool,
              rope_scale: float, rope_theta: float, llama31: dict | None) -> tuple[torch.Tensor, torch.Tensor]:
    """(rows, bound before rounding) of x ``[tokens, heads, head_dim]``, both in 64 bits.

    ``bound``: how far fp32 arithmetic may be off.  The mean is a sum of D squares (relative error at most
    (D + 2) 2^-24, half of it in the root), root, weight and products add 4 roundings, cos and sin are off by
    at most 2^-21 (two units of theirs and the rounding of an angle in turns), and each rotated element is two products and
    a sum: (D / 2 + 8) 2^-24 + 2^-20 of the pair's length.
    """
    d = x.shape[-1]
    y = x.double()
    y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * weight.double()
    size = y.abs()
    f = frequencies(rotary_dim, rope_scale, rope_theta, llama31)
    angle = pos.double()[:, None, None] * f
    c, s = torch.cos(angle), torch.sin(angle)
    first, second = ((slice(0, rotary_dim, 2), slice(1, rotary_dim, 2)) if interleave
                     else (slice(0, rotary_dim // 2), slice(rotary_dim // 2, rotary_dim)))
    out = y.clone()
    a, b = y[..., first], y[..., second]
    out[..., first], out[..., second] = a * c - b * s, b * c + a * s
    length = torch.sqrt(a * a + b * b)
    size[..., first], size[..., second] = length, length
    return out, size * ((d / 2 + 8) * 2.0 ** -24 + 2.0 ** -20)


def rounded(out: torch.Tensor, bound: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """The bound with the rounding to ``dtype``: half a step of the value, or of the smallest subnormal."""
    i = torch.finfo(dtype)
    return bound + (out.abs() + bound) * i.eps / 2 + i.smallest_normal * i.eps / 2
