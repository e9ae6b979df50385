"""MXFP4 in 64 bits: what quantisation gives, and what codes and scale bytes stand for."""

from __future__ import annotations

import torch

GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """bf16 [rows, cols] -> (codes [rows, cols / 2] uint8, scale bytes [rows, cols / 32] uint8)."""
    rows, cols = x.shape
    v = x.double().cpu().view(rows, cols // 32, 32)
    amax = v.abs().amax(-1)
    bad = ~torch.isfinite(v).all(-1)
    amax = torch.where(bad, torch.ones_like(amax), amax)
    e = torch.floor(torch.log2(amax.clamp(min=2.0 ** -140))).clamp(min=-125) - 2
    a = (v.abs() / torch.exp2(e)[..., None]).nan_to_num(0.0, 0.0, 0.0)
    grid = torch.tensor(GRID, dtype=torch.float64)
    far = (a[..., None] - grid).abs()
    # the nearest; of two as near, the even code
    best = far.amin(-1, keepdim=True)
    near = far == best
    even = near & (torch.arange(8) % 2 == 0)
    code = torch.where(even.any(-1), even.to(torch.uint8).argmax(-1), near.to(torch.uint8).argmax(-1))
    code = torch.where(bad[..., None], 0, code + 8 * torch.signbit(x.cpu().view(v.shape)))
    byte = torch.where(bad, 255, (e + 127).long())
    code = code.view(rows, cols // 2, 2).to(torch.uint8)
    return code[..., 0] | code[..., 1] << 4, byte.to(torch.uint8)


def values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """What row-major codes and scale bytes stand for, float64 [rows, cols]."""
    codes, scales = codes.cpu(), scales.cpu()
    rows, half = codes.shape
    code = torch.stack((codes & 15, codes >> 4), -1).view(rows, half // 16, 32).long()
    grid = torch.tensor(GRID + tuple(-g for g in GRID), dtype=torch.float64)
    unit = torch.exp2(scales.double() - 127)
    unit = torch.where(scales == 255, torch.nan, unit)
    return (grid[code] * unit[..., None]).view(rows, 2 * half)
