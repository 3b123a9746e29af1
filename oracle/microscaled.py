"""The microscaled formats in 64 bits: quantisation by the definition, values of codes.

A block of 32 elements has the least exponent e with max|x| <= T * 2^e (T = 464 for e4m3,
7 for e2m1: the largest magnitudes that still round to a code), at least -126 and at most
119 or 125 (where every code is still finite in fp32); codes are the nearest representable
x * 2^-e, ties to the even code, the largest beyond it, and the scale byte is e + 127.  A block of zeros has 127, a block with a NaN or an infinity 255 and codes 0.
"""

from __future__ import annotations

import torch

BLOCK = 32
E4M3 = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()  # values of the codes; 127, 255: NaN
E2M1 = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64)
LIMIT = {8: 464.0, 4: 7.0}
HIGHEST = {8: 119, 4: 125}


def _nearest(y: torch.Tensor, bits: int) -> torch.Tensor:
    """Codes nearest to y (|y| within the format's limit), ties to the even code."""
    grid = E4M3[:127] if bits == 8 else E2M1[:8]
    a = y.abs().clamp(max=float(grid[-1])).contiguous()
    hi = torch.searchsorted(grid, a).clamp(max=len(grid) - 1)  # first code at or above a
    lo = (hi - 1).clamp(min=0)
    up, down = grid[hi] - a, a - grid[lo]
    code = torch.where((up < down) | ((up == down) & (hi % 2 == 0)) | (grid[hi] == a), hi, lo)
    return code + torch.signbit(y).long() * (128 if bits == 8 else 8)


def quantize(x: torch.Tensor, bits: int) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of x ``[..., n]``: uint8 codes ``[..., n]`` (one per element) and scale bytes ``[..., n / 32]``."""
    b = x.double().reshape(*x.shape[:-1], -1, BLOCK)
    peak = b.abs().amax(-1)
    bad = ~torch.isfinite(b).all(-1)
    peak = torch.where(bad, 0.0, peak)
    e = torch.full(peak.shape, -126.0, dtype=torch.float64)
    for _ in range(260):
        more = (peak > LIMIT[bits] * torch.exp2(e)) & (e < HIGHEST[bits])
        if not more.any():
            break
        e = e + more
    scales = torch.where(peak == 0, 127, e.long() + 127)
    codes = _nearest(torch.where(bad[..., None], 0.0, b) / torch.exp2(scales.double() - 127)[..., None], bits)
    scales = torch.where(bad, 255, scales)
    codes = torch.where(bad[..., None], 0, codes)
    return codes.reshape(x.shape).to(torch.uint8), scales.to(torch.uint8)


def values(codes: torch.Tensor, scales: torch.Tensor, bits: int) -> torch.Tensor:
    """What one-per-element codes and their scale bytes stand for, in 64 bits."""
    v = (E4M3 if bits == 8 else E2M1)[codes.long()].reshape(*codes.shape[:-1], -1, BLOCK)
    s = torch.exp2(scales.double() - 127)
    return torch.where((scales == 255)[..., None], float("nan"), v * s[..., None]).reshape(codes.shape)


def pack(codes: torch.Tensor, bits: int) -> torch.Tensor:
    """One-per-element codes as the cache's bytes (4 bits: the even element in the low half)."""
    return codes if bits == 8 else codes[..., 0::2] | (codes[..., 1::2] << 4)


def unpack(rows: torch.Tensor, bits: int) -> torch.Tensor:
    return rows if bits == 8 else torch.stack([rows & 15, rows >> 4], -1).flatten(-2)
