"""Microscaled 4-bit floating point (MXFP4): matrices, quantisation and linear layers.

A block of 32 values of a row shares a power of two and each value is one of
0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign (OCP Microscaling Formats v1.0): 4.25
bits per value.  ``MXFP4`` holds a matrix [rows, cols], cols a multiple of 32, in
the matrix instructions' operand order; ``quantize_mxfp4(x)`` makes one of bf16 rows,
``MXFP4.from_codes`` of a checkpoint's row-major codes and scale bytes.

``linear_mxfp4(x, weight, bias)`` is ``x @ weight.T + bias`` with an MXFP4 weight;
x bf16, or MXFP4 too.  ``linear_silu_mxfp4(x, gate_up)`` is
``silu(x @ gate.T) * (x @ up.T)`` of a fused gate and up weight in the same launch.
Both accumulate in fp32 and round once.  There is no torch fallback and no backward
pass: tensors that ask for gradients or carry forward-mode tangents are refused.
"""

from __future__ import annotations

import functools

import torch
from torch.autograd import forward_ad

from ._util import SILU, SILU_SUMS, bytes_on, call_on, refuse_derivatives, require_dtype, require_gpu, sums_out

BLOCK = 32
_TILE_ROWS, _SLAB, _TILE_BYTES, _QUAD_BYTES = 16, 128, 1024, 256
_FEW_ROWS = 16  # no call of up to so many rows takes a workspace


def _rows_of(name: str, t: torch.Tensor) -> tuple[int, int]:
    require_gpu(name, t)
    require_dtype(name, t, torch.bfloat16)
    shape = t.shape
    if len(shape) != 2 or t.stride(1) != 1:
        raise ValueError(f"{name} must be [rows, width] with a contiguous last axis; got {tuple(shape)}")
    if t.requires_grad or forward_ad._current_level >= 0:
        refuse_derivatives(name, t)
    return shape


def _out(out: torch.Tensor | None, rows: int, cols: int, like: torch.Tensor) -> torch.Tensor:
    if out is None:
        return torch.empty(rows, cols, dtype=torch.bfloat16, device=like.device)
    if _rows_of("out", out) != (rows, cols) or out.device != like.device:
        raise ValueError(f"out must be [{rows}, {cols}] on {like.device}; got {tuple(out.shape)} on {out.device}")
    return out


class MXFP4:
    """A matrix of microscaled 4-bit floats on a GPU, in operand order."""

    __slots__ = ("rows", "cols", "device", "buffer", "codes_ptr", "scales_ptr")

    def __init__(self, rows: int, cols: int, device):
        """Room for [rows, cols]; its contents are undefined until they are written."""
        if rows < 0 or rows > 1 << 31 or cols <= 0 or cols % BLOCK or cols > 1 << 20:
            raise ValueError(f"an MXFP4 matrix has up to 2^31 rows, columns in blocks of {BLOCK}, at most 2^20; got "
                             f"[{rows}, {cols}]")
        self.rows, self.cols = rows, cols
        tiles = -(-rows // _TILE_ROWS)
        # one allocation (two cost 1.1 us more per call): the codes, then the scales
        codes = tiles * -(-cols // _SLAB) * _TILE_BYTES
        self.buffer = torch.empty(codes + tiles * -(-cols // (4 * _SLAB)) * _QUAD_BYTES, dtype=torch.uint8, device=device)
        self.device = self.buffer.device
        self.codes_ptr = self.buffer.data_ptr()
        self.scales_ptr = self.codes_ptr + codes

    @property
    def shape(self) -> tuple[int, int]:
        return self.rows, self.cols

    @property
    def nbytes(self) -> int:
        return self.buffer.numel()

    @classmethod
    def from_codes(cls, codes: torch.Tensor, scales: torch.Tensor) -> "MXFP4":
        """From row-major codes [rows, cols / 2] (the even column in a byte's lower
        half) and scale bytes [rows, cols / 32], both uint8.  Every scale byte is kept;
        bf16 holds values of 2^128 and up (bytes 253 and 254) as infinities, in
        ``dequantize`` and beside bf16 rows."""
        _check_codes(codes, scales)
        m = cls(codes.shape[0], 2 * codes.shape[1], codes.device)
        call_on(codes, "mi_mxfp4_pack", codes.data_ptr(), scales.data_ptr(), m.codes_ptr, m.scales_ptr,
                m.rows, m.cols)
        return m

    def to_codes(self) -> tuple[torch.Tensor, torch.Tensor]:
        """Row-major codes and scale bytes, as ``from_codes`` takes them."""
        codes = torch.empty(self.rows, self.cols // 2, dtype=torch.uint8, device=self.device)
        scales = torch.empty(self.rows, self.cols // BLOCK, dtype=torch.uint8, device=self.device)
        call_on(codes, "mi_mxfp4_unpack", self.codes_ptr, self.scales_ptr, codes.data_ptr(),
                scales.data_ptr(), self.rows, self.cols)
        return codes, scales

    def dequantize(self, out: torch.Tensor | None = None) -> torch.Tensor:
        """The values as bf16 [rows, cols], exactly."""
        out = _out(out, self.rows, self.cols, self.buffer)
        call_on(out, "mi_mxfp4_dequantize", self.codes_ptr, self.scales_ptr, out.data_ptr(),
                out.stride(0), self.rows, self.cols)
        return out


def _check_codes(codes: torch.Tensor, scales: torch.Tensor) -> None:
    for name, t in (("codes", codes), ("scales", scales)):
        require_gpu(name, t)
        require_dtype(name, t, torch.uint8)
        if t.dim() != 2 or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous matrix; got {tuple(t.shape)}")
    if codes.device != scales.device:
        raise ValueError(f"codes on {codes.device}, scales on {scales.device}")
    if codes.shape[1] == 0 or codes.shape[1] % 16 or scales.shape != (codes.shape[0], codes.shape[1] // 16):
        raise ValueError(f"codes [rows, cols / 2] and scales [rows, cols / 32] expected; got {tuple(codes.shape)} and "
                         f"{tuple(scales.shape)}")


def quantize_mxfp4(x: torch.Tensor, out: MXFP4 | None = None) -> MXFP4:
    """bf16 rows in MXFP4: per block of 32 the power of two that brings its largest
    magnitude into [4, 8), each value the nearest code (ties to even, at most 6).  A
    block with an infinity or a NaN becomes NaN."""
    rows, cols = _rows_of("x", x)
    if out is None:
        out = MXFP4(rows, cols, x.device)
    elif out.shape != (rows, cols) or out.device != x.device:
        raise ValueError(f"out must be [{rows}, {cols}] on {x.device}; got {out.shape} on {out.device}")
    call_on(x, "mi_mxfp4_quantize", x.data_ptr(), x.stride(0), out.codes_ptr, out.scales_ptr, rows, cols)
    return out


def _linear(x, weight: MXFP4, bias, out, silu: int) -> torch.Tensor:
    if not isinstance(weight, MXFP4):
        raise TypeError("the weight must be an MXFP4 matrix")
    n = weight.rows
    if silu:
        if n % 2:
            raise ValueError(f"gate_up must have an even number of rows; got {n}")
        n //= 2
    if isinstance(x, MXFP4):
        rows, k = x.rows, x.cols
        data, scales, stride, like = x.codes_ptr, x.scales_ptr, 0, x.buffer
    else:
        rows, k = _rows_of("x", x)
        data, scales, stride, like = x.data_ptr(), None, x.stride(0), x
    if k != weight.cols:
        raise ValueError(f"x has {k} columns, the weight {weight.cols}")
    if like.device != weight.device:
        raise ValueError(f"x on {like.device}, the weight on {weight.device}")
    if bias is not None:
        require_gpu("bias", bias)
        require_dtype("bias", bias, torch.bfloat16)
        if bias.shape != (n,) or not bias.is_contiguous() or bias.device != like.device:
            raise ValueError(f"bias must be a contiguous [{n}] tensor on {like.device}")
        if bias.requires_grad or forward_ad._current_level >= 0:
            refuse_derivatives("bias", bias)
    out = sums_out(out, rows, n, like.device) if silu == SILU_SUMS else _out(out, rows, n, like)
    if rows and n:
        room = _workspace_size(rows, n, k, silu != 0, scales is not None, like.get_device()) if rows > _FEW_ROWS else 0
        # (a tensor of this call's own: calls on several streams and in graphs share nothing)
        workspace = torch.empty(room, dtype=torch.uint8, device=like.device) if room else None
        call_on(like, "mi_linear_mxfp4", data, stride, scales, weight.codes_ptr, weight.scales_ptr,
                bias.data_ptr() if bias is not None else None, out.data_ptr(), out.stride(0), rows, n, k,
                silu, workspace.data_ptr() if room else None, room)
    return out


@functools.lru_cache(maxsize=4096)
def _workspace_size(rows: int, n: int, k: int, silu: bool, x_mxfp4: bool, device: int | None = None) -> int:
    return bytes_on(device, "mi_linear_mxfp4_workspace_size", rows, n, k, silu, x_mxfp4)


def linear_mxfp4(x: torch.Tensor | MXFP4, weight: MXFP4, bias: torch.Tensor | None = None,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """``x @ weight.T + bias`` as bf16 [rows, n]; x is bf16 [rows, k] or MXFP4.  An out
    that overlaps x, the weight or the bias is refused (columns of one buffer need not)."""
    return _linear(x, weight, bias, out, 0)


def linear_silu_mxfp4(x: torch.Tensor | MXFP4, gate_up: MXFP4, out: torch.Tensor | None = None) -> torch.Tensor:
    """``silu(x @ gate.T) * (x @ up.T)``, gate and up the halves of gate_up's rows."""
    return _linear(x, gate_up, None, out, SILU)


def gate_up_mxfp4(x: torch.Tensor | MXFP4, gate_up: MXFP4, out: torch.Tensor | None = None) -> torch.Tensor:
    """The sums ``x @ gate_up.T`` in fp32 [rows, 2 n], bit for bit those that ``linear_silu_mxfp4`` goes on with: what
    ``adapters.add_adapters_silu`` adds to (n a multiple of 4)."""
    return _linear(x, gate_up, None, out, SILU_SUMS)
