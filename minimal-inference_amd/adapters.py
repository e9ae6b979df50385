"""Low-rank adapters of many requests at once beside a shared projection.

``Adapters`` holds the factors of up to 1,023 adapters of one projection: adapter s adds
``scale[s] * B[s] @ (A[s] @ x)`` to the projection's output of the rows that are its own.  The output
may be several pieces with factors of their own (q, k and v of a fused projection).
``AdapterPlan.plan(slot_of_row)`` sorts a batch's rows by adapter on the GPU, once for
all of its layers and projections; ``add_adapters(y, x, adapters, plan)`` adds to y, in place
or into ``out``, in one or two launches; ``add_adapters_silu``
ends in SiLU(gate) * up, the down projection's input.  x is bf16 rows or an ``mxfp8.MXFP8`` matrix.  Sums are
fp32, rounded once.  There is no backward pass: tensors that ask for gradients or carry
forward-mode tangents are refused.
"""

from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib
from ._util import SILU, SILU_STEPS, SILU_SUMS, bytes_on, call_on, refuse_derivatives, require_dtype, require_gpu, require_i32_vector
from .mxfp8 import MXFP8, _out, _rows8, _rows_of

MAX_SLOTS = 1023
MAX_RANK = 128
MAX_PIECES = 8


def _check_sizes(slots: int, k: int, pieces, rank: int) -> None:
    if not 1 <= slots <= MAX_SLOTS:
        raise ValueError(f"{slots} adapters (1..{MAX_SLOTS})")
    if k <= 0 or k % 32 or k > 1 << 20:
        raise ValueError(f"k is {k}: multiples of 32 up to 2^20")
    if rank <= 0 or rank % 8 or rank > MAX_RANK:
        raise ValueError(f"rank is {rank}: multiples of 8 up to {MAX_RANK} (smaller adapters are padded with zeros)")
    if not 1 <= len(pieces) <= MAX_PIECES or any(n <= 0 or n % 16 or n > 1 << 20 for n in pieces):
        raise ValueError(f"pieces {list(pieces)}: 1 to {MAX_PIECES} multiples of 16 up to 2^20")


class Adapters:
    """Adapters of one projection [k -> sum(pieces)].

    a [slots, len(pieces) * rank, k] and b [slots, sum(pieces), rank] bf16, scale [slots] fp32,
    contiguous and held, not copied.  Piece i's rows of A are [i * rank, (i + 1) * rank)."""

    __slots__ = ("a", "b", "scale", "pieces", "slots", "rank", "k", "n", "device", "columns", "columns_ptr")

    def __init__(self, a: torch.Tensor, b: torch.Tensor, scale: torch.Tensor, pieces):
        pieces = [int(n) for n in pieces]
        for name, t, dtype in (("a", a, torch.bfloat16), ("b", b, torch.bfloat16), ("scale", scale, torch.float32)):
            require_gpu(name, t)
            require_dtype(name, t, dtype)
            refuse_derivatives(name, t)
            if not t.is_contiguous() or t.data_ptr() % 16:
                raise ValueError(f"{name} must be contiguous and 16-byte aligned")
            if t.device != a.device:
                raise ValueError(f"{name} on {t.device}, a on {a.device}")
        if a.dim() != 3 or b.dim() != 3:
            raise ValueError(f"a [slots, pieces * rank, k] and b [slots, n, rank] expected; got {tuple(a.shape)} and {tuple(b.shape)}")
        slots, rank, k = a.shape[0], b.shape[2], a.shape[2]
        _check_sizes(slots, k, pieces, rank)
        if a.shape[1] != len(pieces) * rank or b.shape[:2] != (slots, sum(pieces)) or scale.shape != (slots,):
            raise ValueError(f"a [slots, {len(pieces)} * rank, k], b [slots, {sum(pieces)}, rank] and scale [slots] expected; got "
                             f"{tuple(a.shape)}, {tuple(b.shape)} and {tuple(scale.shape)}")
        self.a, self.b, self.scale, self.pieces = a, b, scale, pieces
        self.slots, self.rank, self.k, self.n, self.device = slots, rank, k, sum(pieces), a.device
        self.columns = (ctypes.c_int32 * len(pieces))(*pieces)
        self.columns_ptr = ctypes.addressof(self.columns)

    @property
    def nbytes(self) -> int:
        return self.a.nbytes + self.b.nbytes + self.scale.nbytes

    @classmethod
    def empty(cls, slots: int, k: int, pieces, rank: int, device) -> "Adapters":
        """Room for so many adapters that add nothing until they are set."""
        pieces = [int(n) for n in pieces]
        _check_sizes(slots, k, pieces, rank)
        bf16 = {"dtype": torch.bfloat16, "device": device}
        return cls(torch.zeros(slots, len(pieces) * rank, k, **bf16), torch.zeros(slots, sum(pieces), rank, **bf16),
                   torch.zeros(slots, dtype=torch.float32, device=device), pieces)

    def set(self, slot: int, factors, scale: float) -> None:
        """Adapter ``slot``: per piece (A [r, k], B [n, r]) with r up to the rank, or None for a piece that
        it leaves alone.  On the current stream; runs in flight elsewhere must not read the slot."""
        if not 0 <= slot < self.slots:
            raise ValueError(f"slot {slot} of {self.slots}")
        factors = list(factors)
        if len(factors) != len(self.pieces):
            raise ValueError(f"factors of {len(factors)} pieces, {len(self.pieces)} expected")
        for n, f in zip(self.pieces, factors):
            if f is not None:
                r = f[0].shape[0]
                if r > self.rank or tuple(f[0].shape) != (r, self.k) or tuple(f[1].shape) != (n, r):
                    raise ValueError(f"A [r, {self.k}] and B [{n}, r], r at most {self.rank}, expected; got "
                                     f"{tuple(f[0].shape)} and {tuple(f[1].shape)}")
        with torch.no_grad():
            self.a[slot].zero_()
            self.b[slot].zero_()
            column = 0
            for i, (n, f) in enumerate(zip(self.pieces, factors)):
                if f is not None:
                    r = f[0].shape[0]
                    self.a[slot, i * self.rank: i * self.rank + r].copy_(f[0])
                    self.b[slot, column: column + n, :r].copy_(f[1])
                column += n
            self.scale[slot] = float(scale)

    def clear(self, slot: int) -> None:
        """Adapter ``slot`` adds nothing from here on."""
        self.set(slot, [None] * len(self.pieces), 0.0)


class AdapterPlan:
    """The rows of a batch sorted by adapter.  Runs read the last plan made before them on their stream;
    a captured graph reads the buffer as it is when it is replayed, for the rows that it was captured with
    (after a plan of another number of rows its outputs are NaN)."""

    __slots__ = ("buffer", "slots", "max_rows", "rows", "device")

    def __init__(self, max_rows: int, slots: int, device):
        size = int(_lib.load().mi_adapter_plan_size(max_rows, slots))
        if size == 0:
            raise ValueError(f"{max_rows} rows (0..2^22), {slots} adapters (1..{MAX_SLOTS})")
        self.buffer = torch.zeros(size, dtype=torch.uint8, device=device)  # (no tiles)
        self.device = self.buffer.device
        self.slots, self.max_rows, self.rows = slots, max_rows, 0

    def plan(self, slot_of_row: torch.Tensor) -> None:
        """slot_of_row [rows] int32 on the GPU: each row's adapter; -1, or any other number outside
        0..slots - 1, for none."""
        require_i32_vector("slot_of_row", slot_of_row)
        rows = slot_of_row.shape[0]
        if rows > self.max_rows or slot_of_row.device != self.device:
            raise ValueError(f"slot_of_row has {rows} rows on {slot_of_row.device}; up to {self.max_rows} on {self.device}")
        call_on(self.buffer, "mi_adapter_plan", self.buffer.data_ptr(), self.buffer.numel(), slot_of_row.data_ptr(), rows,
                self.slots)
        self.rows = rows


@functools.lru_cache(maxsize=4096)
def _workspace_size(rows: int, slots: int, k: int, rank: int, pieces: int, n: int, silu: bool, device: int | None = None) -> int:
    return bytes_on(device, "mi_add_adapters_workspace_size", rows, slots, k, rank, pieces, n, silu)


def _sums_of(y: torch.Tensor) -> tuple[int, int]:
    refuse_derivatives("y", y)
    if y.dim() != 2 or y.stride(1) != 1:
        raise ValueError(f"y must be [rows, width] with a contiguous last axis; got {tuple(y.shape)}")
    return y.shape


def _add(y, x, adapters, plan, out, silu: int, quantize: bool):
    if silu == SILU and y.dtype == torch.float32 and y.is_cuda:
        silu = SILU_SUMS
    rows, n = _sums_of(y) if silu == SILU_SUMS else _rows_of("y", y)
    device = y.device
    if not isinstance(adapters, Adapters) or not isinstance(plan, AdapterPlan):
        raise TypeError("adapters must be an Adapters and plan an AdapterPlan")
    if isinstance(x, MXFP8):
        data, stride, scales, s_stride, shape, at = x.codes_ptr, x.codes_stride, x.scales_ptr, x.scales_stride, x.shape, x.device
    else:
        shape = _rows_of("x", x)
        data, stride, scales, s_stride, at = x.data_ptr(), x.stride(0), None, 0, x.device
    if (n, tuple(shape)) != (adapters.n, (rows, adapters.k)):
        raise ValueError(f"y [rows, {adapters.n}] and x [rows, {adapters.k}] expected; got {(rows, n)} and {tuple(shape)}")
    if plan.rows != rows or plan.slots != adapters.slots:
        raise ValueError(f"the plan is of {plan.rows} rows and {plan.slots} adapters, the call of {rows} and {adapters.slots}")
    if not device == at == adapters.device == plan.device:
        raise ValueError(f"y on {device}, x on {at}, the adapters on {adapters.device}, the plan on {plan.device}")
    if silu and (len(adapters.pieces) != 2 or adapters.pieces[0] != adapters.pieces[1]):
        raise ValueError(f"SiLU is of gate and up, two pieces of as many columns; got {adapters.pieces}")
    out_scales, out_s_stride = None, 0
    if quantize:
        out = _rows8(out, rows, n // 2, device)
        to, out_stride, out_scales, out_s_stride = out.codes_ptr, out.codes_stride, out.scales_ptr, out.scales_stride
    else:
        out = y if out is None and not silu else _out(out, rows, n // 2 if silu else n, device)
        to, out_stride = out.data_ptr(), out.stride(0)
    if rows:
        room = _workspace_size(rows, adapters.slots, adapters.k, adapters.rank, len(adapters.pieces), n, silu != 0, device.index)
        # (a tensor of this call's own: calls on several streams and in graphs share nothing)
        workspace = torch.empty(room, dtype=torch.uint8, device=device) if room else None
        call_on(y, "mi_add_adapters", y.data_ptr(), y.stride(0), data, stride, scales, s_stride, adapters.a.data_ptr(),
                adapters.b.data_ptr(), adapters.scale.data_ptr(), adapters.slots, adapters.k, adapters.rank,
                adapters.columns_ptr, len(adapters.pieces), to, out_stride, out_scales, out_s_stride, plan.buffer.data_ptr(),
                rows, silu, workspace.data_ptr() if room else None, room)
    return out


def add_adapters(y: torch.Tensor, x: torch.Tensor | MXFP8, adapters: Adapters, plan: AdapterPlan,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """``y[t] + scale[s] * B[s] @ (A[s] @ x[t])`` with s row t's adapter in the plan; rows without one are
    y's.  Into ``out``, in place in y when that is not given; an out that overlaps another argument is refused."""
    return _add(y, x, adapters, plan, out, 0, False)


def add_adapters_silu(y: torch.Tensor, x: torch.Tensor | MXFP8, adapters: Adapters, plan: AdapterPlan,
                      out: "torch.Tensor | MXFP8 | None" = None, *, quantize: bool = False,
                      stepwise: bool = False) -> "torch.Tensor | MXFP8":
    """``silu(gate) * up`` of what ``add_adapters`` makes of a fused gate and up projection's y [rows, 2 n], held in
    fp32 up to the one rounding: bf16 [rows, n], or with ``quantize`` MXFP8 (n a multiple of 32).  y is left
    as it is; the adapters have two pieces of n columns.

    Rows without an adapter get the bits that the projection's own gated form leaves them, whatever rows stand beside
    them: with y the fp32 sums of ``mxfp8.gate_up_mxfp8`` and ``quantize`` those of ``linear_silu_mxfp8(...,
    quantize=True)``, with those of ``mxfp4.gate_up_mxfp4`` those of ``linear_silu_mxfp4``, and with ``stepwise``, y the
    bf16 of ``dense.linear``, those of ``dense.linear_silu`` (sum, silu and product each rounded to bf16)."""
    if stepwise and quantize:
        raise ValueError("rows in MXFP8 are rounded once: not stepwise")
    return _add(y, x, adapters, plan, out, SILU_STEPS if stepwise else SILU, quantize)
