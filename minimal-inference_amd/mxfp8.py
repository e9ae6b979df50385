"""Microscaled 8-bit floating point (MXFP8): rows, the norm that leaves them, linear layers.

A block of 32 values of a row shares a power of two and each value is an e4m3 float
(OCP Microscaling Formats v1.0): 8.25 bits per value.  ``MXFP8`` holds a matrix
[rows, cols], cols a multiple of 32, row-major as checkpoints do: ``codes``
(float8_e4m3fn) and scale bytes ``scales`` (uint8, [rows, cols / 32]).
``quantize_mxfp8(x)`` makes one of bf16 rows, ``MXFP8.from_codes`` of a checkpoint's
tensors, ``add_rms_norm_mxfp8`` of the residual stream before a block.

``linear_mxfp8(x, weight, bias)`` is ``x @ weight.T + bias`` and
``linear_silu_mxfp8(x, gate_up)`` is ``silu(x @ gate.T) * (x @ up.T)`` of a fused gate
and up weight, both operands MXFP8; the latter leaves MXFP8 rows again with
``quantize=True``, and ``gate_up_mxfp8(x, gate_up)`` leaves its sums as they are.  Sums are fp32, rounded once, but the matrix instruction cuts each product to a multiple of
2^-13 of the largest of its eight neighbours in k: 1.5e-5 of the result's
norm on normal values, 2.7e-5 where single channels stand out, against 1.7e-3 that the rounding to bf16 makes.
The same call repeats its bits.  There is no torch fallback and no backward pass: tensors that
ask for gradients or carry forward-mode tangents are refused.
"""

from __future__ import annotations

import functools

import torch
from torch.autograd import forward_ad

from ._util import SILU, SILU_SUMS, bytes_on, call_on, refuse_derivatives, require_dtype, require_gpu, sums_out

BLOCK = 32
_PIECE = 16  # bytes of scales that are read together


def _rows_of(name: str, t: torch.Tensor) -> tuple[int, int]:
    require_gpu(name, t)
    require_dtype(name, t, torch.bfloat16)
    shape = t.shape
    if len(shape) != 2 or t.stride(1) != 1:
        raise ValueError(f"{name} must be [rows, width] with a contiguous last axis; got {tuple(shape)}")
    if t.requires_grad or forward_ad._current_level >= 0:
        refuse_derivatives(name, t)
    return shape


def _out(out: torch.Tensor | None, rows: int, cols: int, device) -> torch.Tensor:
    if out is None:
        return torch.empty(rows, cols, dtype=torch.bfloat16, device=device)
    if _rows_of("out", out) != (rows, cols) or out.device != device:
        raise ValueError(f"out must be [{rows}, {cols}] on {device}; got {tuple(out.shape)} on {out.device}")
    return out


class MXFP8:
    """A matrix of microscaled 8-bit floats on a GPU."""

    __slots__ = ("rows", "cols", "device", "codes_ptr", "codes_stride", "scales_ptr", "scales_stride", "_held", "anchor")

    def __init__(self, rows: int, cols: int, device):
        """Room for [rows, cols]; its contents are undefined until they are written."""
        if rows < 0 or rows > 1 << 31 or cols <= 0 or cols % BLOCK or cols > 1 << 20:
            raise ValueError(f"an MXFP8 matrix has up to 2^31 rows, columns in blocks of {BLOCK}, at most 2^20; got "
                             f"[{rows}, {cols}]")
        self.rows, self.cols = rows, cols
        self.codes_stride, self.scales_stride = cols, -(-cols // (_PIECE * BLOCK)) * _PIECE
        # one allocation: the codes, then the scales
        self.anchor = torch.empty(rows * (cols + self.scales_stride), dtype=torch.uint8, device=device)
        self._held = None
        self.device = self.anchor.device
        self.codes_ptr = self.anchor.data_ptr()
        self.scales_ptr = self.codes_ptr + rows * cols

    @classmethod
    def _room(cls, rows: int, cols: int, device) -> "MXFP8":
        """``MXFP8(rows, cols, device)`` of sizes that an entry has checked or will."""
        m = cls.__new__(cls)
        m.rows, m.cols, m.device, m._held = rows, cols, device, None
        m.codes_stride = cols
        stride = m.scales_stride = (cols + 511 >> 9) * _PIECE
        m.anchor = torch.empty(rows * (cols + stride), dtype=torch.uint8, device=device)
        m.codes_ptr = at = m.anchor.data_ptr()
        m.scales_ptr = at + rows * cols
        return m

    @property
    def shape(self) -> tuple[int, int]:
        return self.rows, self.cols

    @property
    def nbytes(self) -> int:
        return self.rows * (self.cols + self.scales_stride)

    @property
    def codes(self) -> torch.Tensor:
        """float8_e4m3fn [rows, cols], no copy."""
        if self._held is not None:
            return self._held[0]
        n = self.rows * self.cols
        return self.anchor[:n].view(torch.float8_e4m3fn).view(self.rows, self.cols)

    @property
    def scales(self) -> torch.Tensor:
        """Scale bytes, uint8 [rows, cols / 32], no copy: the block's power of two is 2^(byte - 127)."""
        if self._held is not None:
            return self._held[1]
        return self.anchor[self.rows * self.cols:].view(self.rows, self.scales_stride)[:, : self.cols // BLOCK]

    @classmethod
    def from_codes(cls, codes: torch.Tensor, scales: torch.Tensor) -> "MXFP8":
        """From codes [rows, cols] (float8_e4m3fn, or their bytes as uint8) and scale bytes
        [rows, cols / 32] (uint8 or float8_e8m0fnu).  The tensors are held, not copied, where their rows
        lie as the kernels read them (codes in whole 16 bytes, a row's scales a multiple of 16), else
        copied."""
        codes, scales = _check_codes(codes, scales)
        rows, cols = codes.shape
        aligned = all(t.data_ptr() % 16 == 0 and t.stride(1) == 1 and (rows == 1 or (t.stride(0) % 16 == 0 and t.stride(0) >= t.shape[1]))
                      for t in (codes, scales))
        if not aligned or scales.shape[1] % _PIECE:
            m = cls(rows, cols, codes.device)
            m.codes.view(torch.uint8).copy_(codes)
            m.scales.copy_(scales)
            return m
        m = cls.__new__(cls)
        m.rows, m.cols, m.device = rows, cols, codes.device
        m.anchor, m._held = codes, (codes.view(torch.float8_e4m3fn), scales)
        m.codes_ptr, m.codes_stride = codes.data_ptr(), codes.stride(0) if rows > 1 else cols
        m.scales_ptr, m.scales_stride = scales.data_ptr(), scales.stride(0) if rows > 1 else scales.shape[1]
        return m

    def dequantize(self, out: torch.Tensor | None = None) -> torch.Tensor:
        """The values as bf16 [rows, cols]: exactly, but below 2^-133."""
        out = _out(out, self.rows, self.cols, self.device)
        call_on(out, "mi_mxfp8_dequantize", self.codes_ptr, self.codes_stride, self.scales_ptr, self.scales_stride,
                out.data_ptr(), out.stride(0), self.rows, self.cols)
        return out


def _check_codes(codes: torch.Tensor, scales: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Both as bytes."""
    for name, t, types in (("codes", codes, (torch.float8_e4m3fn, torch.uint8)),
                           ("scales", scales, (torch.uint8, torch.float8_e8m0fnu))):
        require_gpu(name, t)
        if t.dtype not in types:
            raise ValueError(f"{name} must be {types[0]} or {types[1]} (got {t.dtype})")
        refuse_derivatives(name, t)
        if t.dim() != 2:
            raise ValueError(f"{name} must be a matrix; got {tuple(t.shape)}")
    if codes.device != scales.device:
        raise ValueError(f"codes on {codes.device}, scales on {scales.device}")
    if codes.shape[1] == 0 or codes.shape[1] % BLOCK or scales.shape != (codes.shape[0], codes.shape[1] // BLOCK):
        raise ValueError(f"codes [rows, cols] and scales [rows, cols / 32] expected; got {tuple(codes.shape)} and "
                         f"{tuple(scales.shape)}")
    if codes.shape[0] > 1 << 31 or codes.shape[1] > 1 << 20:
        raise ValueError(f"an MXFP8 matrix has up to 2^31 rows and 2^20 columns; got {tuple(codes.shape)}")
    return codes.view(torch.uint8), scales.view(torch.uint8)


def _rows8(out: "MXFP8 | None", rows: int, cols: int, device) -> MXFP8:
    if out is None:
        if cols % BLOCK or cols <= 0 or cols > 1 << 20:
            raise ValueError(f"an MXFP8 matrix has columns in blocks of {BLOCK}, at most 2^20; got [{rows}, {cols}]")
        return MXFP8._room(rows, cols, device)
    if not isinstance(out, MXFP8) or out.shape != (rows, cols) or out.device != device:
        raise ValueError(f"out must be an MXFP8 matrix [{rows}, {cols}] on {device}")
    return out


def quantize_mxfp8(x: torch.Tensor, out: MXFP8 | None = None) -> MXFP8:
    """bf16 rows in MXFP8: per block of 32 the least power of two that keeps all of it within
    448, each value the nearest code (ties to even).  A block with an infinity or a NaN becomes NaN."""
    rows, cols = _rows_of("x", x)
    out = _rows8(out, rows, cols, x.device)
    call_on(x, "mi_mxfp8_quantize", x.data_ptr(), x.stride(0), out.codes_ptr, out.codes_stride, out.scales_ptr,
            out.scales_stride, rows, cols)
    return out


def add_rms_norm_mxfp8(x: torch.Tensor, delta: torch.Tensor | None, weight: torch.Tensor, eps: float, *,
                       x_out: torch.Tensor | None = None, out: MXFP8 | None = None) -> MXFP8:
    """``dense.add_rms_norm`` with its norm in 8 bits: ``x + delta`` rounded to bf16 (into ``x_out``,
    in place in ``x`` when that is not given; without ``delta`` x itself, which is then not written),
    and its ``rms_norm(...) * weight``, quantised as its exact value would be (blocks past fp32's range become NaN).
    Outputs that overlap each other, the weight or another row's input are refused."""
    shape, grad = x.shape, torch.is_grad_enabled()
    if len(shape) != 2:
        raise ValueError(f"x must be [rows, hidden]; got {tuple(shape)}")
    rows, hidden = shape
    if hidden > 16384:  # (the entry takes 32 bits of it)
        raise ValueError(f"hidden is {hidden}: multiples of {BLOCK} up to 16384")
    at, device = x.get_device(), x.device
    if (x.dtype != torch.bfloat16 or at < 0 or x.stride(1) != 1 or (grad and x.requires_grad)):
        _rows_of("x", x)
    for name, t in (("delta", delta), ("x_out", x_out)):
        if t is not None and (t.shape != shape or t.dtype != torch.bfloat16 or t.get_device() != at or t.stride(1) != 1
                              or (grad and t.requires_grad)):
            _rows_of(name, t)
            raise ValueError(f"{name} must be [{rows}, {hidden}] on {device}; got {tuple(t.shape)} on {t.device}")
    if (weight.shape != (hidden,) or weight.dtype != torch.bfloat16 or weight.get_device() != at or weight.stride(0) != 1
            or (grad and weight.requires_grad)):
        refuse_derivatives("weight", weight)
        raise ValueError(f"weight must be a contiguous bfloat16 [{hidden}] tensor on {device}; got {tuple(weight.shape)} "
                         f"{weight.dtype} on {weight.device}")
    if forward_ad._current_level >= 0:
        for name, t in (("x", x), ("delta", delta), ("weight", weight), ("x_out", x_out)):
            refuse_derivatives(name, t)
    if x_out is None and delta is not None:
        x_out = x
    out = _rows8(out, rows, hidden, device)
    call_on(x, "mi_add_rms_norm_mxfp8", x.data_ptr(), x.stride(0), delta.data_ptr() if delta is not None else None,
            delta.stride(0) if delta is not None else 0, weight.data_ptr(), x_out.data_ptr() if x_out is not None else None,
            x_out.stride(0) if x_out is not None else 0, out.codes_ptr, out.codes_stride, out.scales_ptr,
            out.scales_stride, rows, hidden, eps)
    return out


@functools.lru_cache(maxsize=4096)
def _workspace_size(rows: int, n: int, k: int, silu: bool, device: int | None = None) -> int:
    return bytes_on(device, "mi_linear_mxfp8_workspace_size", rows, n, k, silu)


def _linear(x: MXFP8, weight: MXFP8, bias, out, silu: int, quantize: bool):
    if not isinstance(x, MXFP8) or not isinstance(weight, MXFP8):
        raise TypeError("x and the weight must be MXFP8 matrices (quantize_mxfp8 makes one of bf16 rows)")
    rows, k, n, device = x.rows, x.cols, weight.rows, x.device
    if silu:
        if n % 2:
            raise ValueError(f"gate_up must have an even number of rows; got {n}")
        n //= 2
    if k != weight.cols:
        raise ValueError(f"x has {k} columns, the weight {weight.cols}")
    if device != weight.device:
        raise ValueError(f"x on {device}, the weight on {weight.device}")
    if bias is not None:
        require_gpu("bias", bias)
        require_dtype("bias", bias, torch.bfloat16)
        if bias.shape != (n,) or not bias.is_contiguous() or bias.device != device:
            raise ValueError(f"bias must be a contiguous [{n}] tensor on {device}")
        if bias.requires_grad or forward_ad._current_level >= 0:
            refuse_derivatives("bias", bias)
    if quantize:
        out = _rows8(out, rows, n, device)
        to, stride, scales, s_stride = out.codes_ptr, out.codes_stride, out.scales_ptr, out.scales_stride
    else:
        out = sums_out(out, rows, n, device) if silu == SILU_SUMS else _out(out, rows, n, device)
        to, stride, scales, s_stride = out.data_ptr(), out.stride(0), None, 0
    if rows and n:
        room = _workspace_size(rows, n, k, silu != 0, device.index)
        # (a tensor of this call's own: calls on several streams and in graphs share nothing)
        workspace = torch.empty(room, dtype=torch.uint8, device=device) if room else None
        call_on(x.anchor, "mi_linear_mxfp8", x.codes_ptr, x.codes_stride, x.scales_ptr, x.scales_stride,
                weight.codes_ptr, weight.codes_stride, weight.scales_ptr, weight.scales_stride,
                bias.data_ptr() if bias is not None else None, to, stride, scales, s_stride, rows, n, k, silu,
                workspace.data_ptr() if room else None, room)
    return out


def linear_mxfp8(x: MXFP8, weight: MXFP8, bias: torch.Tensor | None = None,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """``x @ weight.T + bias`` as bf16 [rows, n].  An out that overlaps x, the weight or
    the bias is refused."""
    return _linear(x, weight, bias, out, 0, False)


def linear_silu_mxfp8(x: MXFP8, gate_up: MXFP8, out: "torch.Tensor | MXFP8 | None" = None, *,
                      quantize: bool = False) -> "torch.Tensor | MXFP8":
    """``silu(x @ gate.T) * (x @ up.T)``, gate and up the halves of gate_up's rows, as bf16
    [rows, n], or with ``quantize`` as MXFP8, rounded from fp32 (n a multiple of 32; silu within 2^-20)."""
    if quantize and isinstance(gate_up, MXFP8) and gate_up.rows // 2 % BLOCK:
        raise ValueError(f"rows in MXFP8 have columns in blocks of {BLOCK}; got {gate_up.rows // 2}")
    return _linear(x, gate_up, None, out, SILU, quantize)


def gate_up_mxfp8(x: MXFP8, gate_up: MXFP8, out: torch.Tensor | None = None) -> torch.Tensor:
    """The sums ``x @ gate_up.T`` in fp32 [rows, 2 n], bit for bit those of which ``linear_silu_mxfp8`` makes MXFP8
    rows: what ``adapters.add_adapters_silu`` adds to (n a multiple of 4)."""
    return _linear(x, gate_up, None, out, SILU_SUMS, False)
