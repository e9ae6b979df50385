"""Fused batched sampler -- drop-in for the reference's ``sample_batch`` /
``sample`` (scheduler.py:310-343), plus top-p.

``sample_batch(logits [B, S, V], temperatures)`` keeps the reference's
contract: temperatures are rounded to the logits dtype (bf16), rows with
temperature <= 0 are greedy (argmax, first index on ties), the rest draw one
token from softmax(logits / t) in fp32.  One fused kernel per call replaces
softmax + multinomial + argmax + masked index-put; the only host sync is the
final ``.tolist()``, as in the reference.

``Sampler`` is the allocation-free form for graph capture: it owns device
buffers for per-row temperature / top-p, the output ids, the Philox counter
and the kernels' workspaces, one of ``sample`` and one of ``draw`` (sized at
construction for ``vocab`` when given, else for the largest vocabulary seen, which
takes one call before a capture; a workspace that grows is replaced but kept alive,
so a graph captured with the old one never writes into freed memory), so a captured
decode step can include the draw.

``Sampler.draw`` draws from given uniform numbers, one per row, with top-k and min-p
beside temperature and top-p (``set_params(top_k=, min_p=)``): the same numbers give
the same ids on any run.  ``sample_batch`` takes it when it is given ``top_k``,
``min_p`` or ``uniforms``.
"""

from __future__ import annotations

import torch

from . import _lib
from ._util import call_on, require_dtype, require_gpu, stream_of

_DEFAULT_SEED = 0x6D69616D64  # "miamd"
_DRAW_MAX_VOCAB = 1 << 20


class Sampler:
    """Per-device sampler state: rng counter and reusable row buffers."""

    def __init__(self, device: torch.device, max_batch: int, seed: int = _DEFAULT_SEED, vocab: int | None = None):
        self.device = torch.device(device)
        self.max_batch = max_batch
        self.seed = int(seed) & 0xFFFFFFFFFFFFFFFF
        self.rng_offset = torch.zeros(1, dtype=torch.int64, device=self.device)
        self.temperature = torch.zeros(max_batch, dtype=torch.float32, device=self.device)
        self.top_p = torch.ones(max_batch, dtype=torch.float32, device=self.device)
        self.top_k = torch.zeros(max_batch, dtype=torch.int32, device=self.device)
        self.min_p = torch.zeros(max_batch, dtype=torch.float32, device=self.device)
        self._filtered = False  # whether top_k / min_p hold anything but "off"
        self.out = torch.zeros(max_batch, dtype=torch.int64, device=self.device)
        self.draw_workspace = torch.zeros(0, dtype=torch.uint8, device=self.device)
        self.workspace = torch.zeros(0, dtype=torch.uint8, device=self.device)
        self._retired: list[torch.Tensor] = []  # replaced workspaces a captured graph may still use
        if vocab is not None:
            self._workspace_for(vocab)
            self._draw_workspace_for(vocab)

    def _workspace_for(self, vocab: int) -> torch.Tensor:
        need = int(_lib.load().mi_sample_workspace_size(self.max_batch, vocab))
        if self.workspace.numel() < need:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError(f"sampler workspace for vocab {vocab} must be sized before graph capture")
            if self.workspace.numel():
                self._retired.append(self.workspace)
            self.workspace = torch.zeros(need, dtype=torch.uint8, device=self.device)  # counters start at zero
        return self.workspace

    def _draw_workspace_for(self, vocab: int) -> torch.Tensor:
        need = int(_lib.load().mi_draw_workspace_size(self.max_batch, vocab))
        if self.draw_workspace.numel() < need:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError(f"draw workspace for vocab {vocab} must be sized before graph capture")
            if self.draw_workspace.numel():
                self._retired.append(self.draw_workspace)
            self.draw_workspace = torch.empty(need, dtype=torch.uint8, device=self.device)
        return self.draw_workspace

    def set_params(self, temperatures, top_p=None, *, top_k=None, min_p=None) -> None:
        """Copy per-row parameters in (asynchronous host->device copies).  ``top_k`` (0:
        off) and ``min_p`` (0: off) are read by ``draw`` alone."""
        n = len(temperatures)
        if n > self.max_batch:
            raise ValueError(f"{n} rows exceed the sampler's max_batch {self.max_batch}")
        t = torch.as_tensor(temperatures, dtype=torch.float32)
        self.temperature[:n].copy_(t, non_blocking=True)
        if top_p is None:
            self.top_p[:n].fill_(1.0)
        else:
            self.top_p[:n].copy_(torch.as_tensor(top_p, dtype=torch.float32), non_blocking=True)
        filtered = top_k is not None or min_p is not None
        if filtered or self._filtered:
            for buffer, values in ((self.top_k, top_k), (self.min_p, min_p)):
                if values is None:
                    buffer.zero_()
                else:
                    buffer[:n].copy_(torch.as_tensor(values, dtype=buffer.dtype), non_blocking=True)
            self._filtered = filtered

    def draw(self, logits: torch.Tensor, uniforms: torch.Tensor, n: int | None = None,
             out: torch.Tensor | None = None) -> torch.Tensor:
        """Ids for rows 0..n-1 of ``logits`` [B, V] (or [B, 1, V]) from ``uniforms``
        (fp32 in [0, 1), one per row) with the rows' temperature, top-k, min-p and top-p.

        With w = exp((l - max l) / t) and tokens ordered by descending logit, then
        ascending id: the first top_k, of them those with w >= min_p, of those the
        shortest prefix whose mass reaches top_p of theirs, always the first; drawn is
        the lowest id whose cumulative kept weight, in order of ids, exceeds u times
        the kept total.  In 64 bits; temperatures are taken as they are (not rounded to
        bf16).  Rows with temperature <= 0, or with no logit above -inf, give argmax.
        A sampler's draws share its workspace: one at a time.
        """
        if logits.dim() == 3:
            logits = logits[:, -1, :]
        require_gpu("logits", logits)
        require_dtype("logits", logits, torch.bfloat16)
        if logits.dim() != 2 or logits.stride(1) != 1:
            raise ValueError("logits must be [B, V] with a contiguous vocab axis")
        if logits.shape[1] > _DRAW_MAX_VOCAB:  # (the entry takes 32 bits of it)
            raise ValueError(f"rows of {logits.shape[1]} tokens: at most {_DRAW_MAX_VOCAB}")
        n = logits.shape[0] if n is None else n
        if not 0 <= n <= min(logits.shape[0], self.max_batch):
            raise ValueError(f"{n} rows: logits have {logits.shape[0]}, the sampler takes {self.max_batch}")
        require_gpu("uniforms", uniforms)
        require_dtype("uniforms", uniforms, torch.float32)
        if uniforms.dim() != 1 or uniforms.shape[0] < n or not uniforms.is_contiguous():
            raise ValueError(f"uniforms must be a contiguous vector of at least {n}; got {tuple(uniforms.shape)}")
        out = self.out if out is None else out
        require_gpu("out", out)
        require_dtype("out", out, torch.int64)
        if out.dim() != 1 or out.shape[0] < n or not out.is_contiguous():
            raise ValueError(f"out must be a contiguous vector of at least {n}; got {tuple(out.shape)}")
        for t in (uniforms, out, self.temperature):
            if t.get_device() != logits.get_device():
                raise ValueError(f"logits on {logits.device}, other arguments on {t.device}")
        if n:
            ws = self._draw_workspace_for(logits.shape[1])
            call_on(logits, "mi_draw", logits.data_ptr(), logits.stride(0), n, logits.shape[1],
                    self.temperature.data_ptr(), self.top_k.data_ptr(), self.top_p.data_ptr(), self.min_p.data_ptr(),
                    uniforms.data_ptr(), out.data_ptr(), ws.data_ptr(), ws.numel())
        return out[:n]

    def sample(self, logits: torch.Tensor, n: int | None = None, out: torch.Tensor | None = None,
               use_top_p: bool = True) -> torch.Tensor:
        """Draw ids for rows 0..n-1 of ``logits`` [B, V] (or [B, 1, V])."""
        if logits.dim() == 3:
            logits = logits[:, -1, :]
        require_gpu("logits", logits)
        require_dtype("logits", logits, torch.bfloat16)
        if logits.dim() != 2 or logits.stride(1) != 1:
            raise ValueError("logits must be [B, V] with a contiguous vocab axis")
        n = logits.shape[0] if n is None else n
        if n > self.max_batch:
            raise ValueError(f"{n} rows exceed the sampler's max_batch {self.max_batch}")
        out = self.out if out is None else out
        ws = self._workspace_for(logits.shape[1])
        _lib.call(
            "mi_sample", logits.data_ptr(), logits.stride(0), n, logits.shape[1],
            self.temperature.data_ptr(), self.top_p.data_ptr() if use_top_p else None,
            self.seed, self.rng_offset.data_ptr(), out.data_ptr(), ws.data_ptr(), ws.numel(), stream_of(logits),
        )
        return out[:n]


_samplers: dict[tuple[int, int], Sampler] = {}


def _sampler_for(device: torch.device, batch: int) -> Sampler:
    key = (device.index or 0, batch)
    s = _samplers.get(key)
    if s is None:
        s = Sampler(device, max(batch, 1))
        _samplers[key] = s
    return s


def sample_batch(logits: torch.Tensor, temperatures: list[float], top_p: list[float] | None = None, *,
                 top_k: list[int] | None = None, min_p: list[float] | None = None,
                 uniforms: torch.Tensor | None = None) -> list[int]:
    """Sample one id per row of ``logits`` [B, S, V] (last position).

    With ``top_k``, ``min_p`` or ``uniforms`` (fp32 on the GPU, one number in [0, 1) per
    row; torch's generator draws them when they are not given) by ``Sampler.draw``."""
    if logits.dim() != 3:
        raise ValueError(f"logits must be [B, S, V]; got {tuple(logits.shape)}")
    b = logits.shape[0]
    if len(temperatures) != b:
        raise ValueError("one temperature per row is required")
    for name, values in (("top_k", top_k), ("min_p", min_p)):
        if values is not None and len(values) != b:
            raise ValueError(f"one {name} per row is required")
    s = _sampler_for(logits.device, b)
    s.set_params(temperatures, top_p, top_k=top_k, min_p=min_p)
    if top_k is None and min_p is None and uniforms is None:
        ids = s.sample(logits[:, -1, :], b, use_top_p=top_p is not None)
    else:
        if uniforms is None:
            uniforms = torch.rand(b, device=logits.device)
        ids = s.draw(logits[:, -1, :], uniforms, b)
    return ids.tolist()


def sample(logits: torch.Tensor, temperature: float, top_p: float | None = None, *, top_k: int | None = None,
           min_p: float | None = None, uniforms: torch.Tensor | None = None) -> int:
    """Single request: logits [1, S, V] -> one id (scheduler.py:310-316)."""
    one = lambda v: None if v is None else [v]  # noqa: E731
    return sample_batch(logits[:1], [temperature], one(top_p), top_k=one(top_k), min_p=one(min_p), uniforms=uniforms)[0]
