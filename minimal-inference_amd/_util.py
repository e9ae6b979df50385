"""Argument checks and stream plumbing shared by the wrappers."""

from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import _lib


def stream_of(t: torch.Tensor) -> int:
    """Raw hipStream_t of torch's current stream on ``t``'s device (the handle itself:
    a ``Stream`` object around it cost each call 1.9 us, this 0.1)."""
    return torch._C._cuda_getCurrentRawStream(t.get_device())


def call_on(t: torch.Tensor, name: str, *args) -> None:
    """``_lib.call`` on ``t``'s device with its current stream as the last argument; the
    current device changes only where it is another (the context manager costs 3 us)."""
    device = t.get_device()
    entry = getattr(_lib.load(), name)
    if device == torch._C._cuda_getDevice():
        status = entry(*args, torch._C._cuda_getCurrentRawStream(device))
    else:
        with torch.cuda.device(device):
            status = entry(*args, torch._C._cuda_getCurrentRawStream(device))
    if status:
        _lib.check(status, name)


def bytes_on(device: int | None, name: str, *args) -> int:
    """What a size entry answers with ``device`` current (its number of CUs decides how work is shared, here as
    in the launch, which ``call_on`` makes on the tensors' device); None: the current one."""
    entry = getattr(_lib.load(), name)
    if device is None or device == torch._C._cuda_getDevice():
        return int(entry(*args))
    with torch.cuda.device(device):
        return int(entry(*args))


def require_gpu(name: str, t: torch.Tensor) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on a GPU (got {t.device}); there is no CPU path")


def require_dtype(name: str, t: torch.Tensor, dtype: torch.dtype) -> None:
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype} (got {t.dtype})")


def refuse_derivatives(name: str, t: torch.Tensor | None) -> None:
    """Of an operator without a backward pass: a tensor that asks for a gradient, or that
    carries a forward-mode tangent (which a kernel of the library would drop)."""
    if t is None:
        return
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient: there is no backward pass")
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        raise ValueError(f"{name} has a forward-mode tangent: there is no derivative")


SILU, SILU_SUMS, SILU_STEPS = 1, 2, 3  # MI_SILU, MI_SILU_SUMS, MI_SILU_STEPS


def sums_out(out: torch.Tensor | None, rows: int, n: int, device) -> torch.Tensor:
    """Room for the fp32 sums of a gated product, gate's n and up's n columns."""
    if n % 4:
        raise ValueError(f"gate and up of a multiple of 4 columns each; got {n}")
    if out is None:
        return torch.empty(rows, 2 * n, dtype=torch.float32, device=device)
    require_gpu("out", out)
    require_dtype("out", out, torch.float32)
    if out.shape != (rows, 2 * n) or out.stride(1) != 1 or out.device != device:
        raise ValueError(f"out must be [{rows}, {2 * n}] with a contiguous last axis on {device}; got {tuple(out.shape)} on {out.device}")
    refuse_derivatives("out", out)
    return out


def require_i32_vector(name: str, t: torch.Tensor) -> None:
    require_gpu(name, t)
    require_dtype(name, t, torch.int32)
    if t.dim() != 1 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous 1-D int32 tensor (got shape {tuple(t.shape)})")


def require_pool(name: str, pool: torch.Tensor) -> tuple[int, int, int, int]:
    """Validate an NHD pool [pages, 2, page_size, kv_heads, head_dim] bf16."""
    require_gpu(name, pool)
    require_dtype(name, pool, torch.bfloat16)
    if pool.dim() != 5 or pool.shape[1] != 2:
        raise ValueError(f"{name} must be [num_pages, 2, page_size, num_kv_heads, head_dim] "
                         f"(NHD); got {tuple(pool.shape)}")
    if not pool.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return tuple(int(x) for x in (pool.shape[0], pool.shape[2], pool.shape[3], pool.shape[4]))


def require_rows(name: str, t: torch.Tensor, heads: int, head_dim: int) -> None:
    """[N, heads, head_dim] bf16 with head_dim contiguous."""
    require_gpu(name, t)
    require_dtype(name, t, torch.bfloat16)
    if t.dim() != 3 or t.shape[1] != heads or t.shape[2] != head_dim:
        raise ValueError(f"{name} must be [N, {heads}, {head_dim}]; got {tuple(t.shape)}")
    if t.stride(2) != 1:
        raise ValueError(f"{name} must have a contiguous last axis")
