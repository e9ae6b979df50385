"""MXFP8 in 64 bits: what quantisation gives, and what codes and scale bytes stand for."""

from __future__ import annotations

import torch

BLOCK = 32
LARGEST = 448.0

# the magnitudes of codes 0 .. 126 (127 is NaN): 2^-9 steps up to 2^-6, then eight to a power of two
GRID = torch.tensor([(c % 8) / 512 if c < 8 else (1 + c % 8 / 8) * 2.0 ** (c // 8 - 7) for c in range(127)],
                    dtype=torch.float64)


def quantize(v: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows [rows, cols] of any float type -> (codes uint8 [rows, cols], scale bytes uint8 [rows, cols / 32])."""
    rows, cols = v.shape
    v = v.double().cpu().view(rows, cols // BLOCK, BLOCK)
    bad = ~torch.isfinite(v).all(-1)
    sign = torch.signbit(v)
    a = torch.where(bad[..., None], 0.0, v.abs())
    amax = a.amax(-1)
    # the least power of two, 2^-127 at least, of which 448 are no less than the largest
    powers = torch.exp2(torch.arange(-127, 128, dtype=torch.float64))
    e = torch.searchsorted(LARGEST * powers, amax.contiguous())  # powers below it are too small
    a = a / powers[e][..., None]
    above = torch.searchsorted(GRID, a.contiguous()).clamp(max=126)
    below = (above - 1).clamp(min=0)
    up, down = GRID[above] - a, a - GRID[below]
    code = torch.where(up < down, above, torch.where(down < up, below, torch.where(above % 2 == 0, above, below)))
    code = torch.where(a == 0, 0, code)
    code = torch.where(bad[..., None], 0, code + 128 * sign)
    return code.view(rows, cols).to(torch.uint8), torch.where(bad, 255, e).to(torch.uint8)


def values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """What codes (bytes) and scale bytes stand for, float64 [rows, cols], where they lie."""
    codes, scales = codes.view(torch.uint8), scales.view(torch.uint8)
    grid = torch.cat([GRID, torch.tensor([torch.nan], dtype=torch.float64)]).to(codes.device)
    grid = torch.cat([grid, -grid])
    unit = torch.where(scales == 255, torch.nan, torch.exp2(scales.double() - 127))
    rows, cols = codes.shape
    return (grid[codes.long()].view(rows, cols // BLOCK, BLOCK) * unit[..., None]).view(rows, cols)
