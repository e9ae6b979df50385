"""Dense Qwen2 / Mistral transformer driving the paged-attention path.

Restates model.py of the reference (ModelConfig 37-71, RoPE 79-107, RMSNorm
115-122, Attention 126-252, MLP 301-311, DecoderLayer 314-344, Model
352-435).  The GEMMs of many rows stay on PyTorch-ROCm (hipBLASLt); the
attention layer calls the HIP library through the reference's drop-in
surface: ``append_paged_kv_cache`` then ``wrapper.run`` (model.py:207-235),
without the reference's Q-head padding (model.py:134-137, 226-243): any
integer GQA group runs natively.

Layout choices (dense path only; numerics match the separate-projection
form): q/k/v projections are one fused GEMM and gate/up one fused GEMM, and
prefill computes logits only for each request's last position.  By default
RoPE on q and k and the K/V append run as one HIP launch
(``rope_append_paged_kv_cache``), bit-identical to the reference's bf16
RoPE ops followed by the append, and in decode steps the attention launch
does both itself (``run_rope_append``; ``fused_decode=False`` keeps the
separate launch), bit-identical again; ``fused_rope=False`` keeps the
separate ops.
By default the residual adds and the RMSNorms that follow them run as one
HIP kernel each (``dense.add_rms_norm``, fp32 math, one bf16 rounding per
output), the projections of a decode step's few rows on the kernel that streams
each weight once (``dense.linear``), SiLU(gate) * up in that launch too or, for
more rows, as a kernel of its own (``dense.linear_silu``);
``fused_dense=False`` keeps torch's ``F.linear``, ``F.rms_norm``, adds and
``F.silu(g) * u``.  ``Model.quantize_weights()`` turns the layers' projections into
microscaled 4-bit matrices (``mxfp4.MXFP4``), which every step then multiplies by
``mxfp4.linear_mxfp4`` / ``linear_silu_mxfp4``, whatever its rows; ``quantize_weights("mxfp8")``
into 8-bit ones (``mxfp8.MXFP8``), whose inputs are 8-bit rows too: the norms leave such rows
(``add_rms_norm_mxfp8``), SiLU(gate) * up does in its projection's launch, and the attention's
outputs are quantised.  ``Model.enable_adapters()`` makes room for low-rank adapters beside the
projections (``adapters.add_adapters``), which the rows of a step take by their backend's
``adapter_plan``.  RoPE tables are held in the model dtype, as the reference's are after ``.to(dtype)``
(server.py:251).  Weights are random-initialised on the device (N(0, 0.02),
norms 1) -- the benchmark configurations use random weights.
"""

from __future__ import annotations

import dataclasses
import gc
import json
import math
import os
import weakref

import torch
import torch.nn.functional as F

from .adapters import Adapters, add_adapters, add_adapters_silu
from .dense import add_rms_norm, linear, linear_silu
from .mxfp4 import BLOCK, MXFP4, gate_up_mxfp4, linear_mxfp4, linear_silu_mxfp4, quantize_mxfp4
from .mxfp8 import MXFP8, add_rms_norm_mxfp8, gate_up_mxfp8, linear_mxfp8, linear_silu_mxfp8, quantize_mxfp8
from .page import append_paged_kv_cache, rope_append_paged_kv_cache


@dataclasses.dataclass
class ModelConfig:
    hidden_size: int = 896
    num_attention_heads: int = 14
    num_key_value_heads: int = 2
    head_dim: int = 64
    num_hidden_layers: int = 24
    intermediate_size: int = 4864
    vocab_size: int = 151936
    rms_norm_eps: float = 1e-6
    rope_theta: float = 1_000_000.0
    max_position_embeddings: int = 32768
    tie_word_embeddings: bool = True
    attn_bias: bool = True

    @classmethod
    def from_pretrained(cls, model_path: str) -> "ModelConfig":
        """Same field mapping as the reference (model.py:52-71)."""
        with open(os.path.join(model_path, "config.json")) as f:
            raw = json.load(f)
        return cls(
            hidden_size=raw["hidden_size"],
            num_attention_heads=raw["num_attention_heads"],
            num_key_value_heads=raw["num_key_value_heads"],
            head_dim=raw.get("head_dim", raw["hidden_size"] // raw["num_attention_heads"]),
            num_hidden_layers=raw["num_hidden_layers"],
            intermediate_size=raw["intermediate_size"],
            vocab_size=raw["vocab_size"],
            rms_norm_eps=raw.get("rms_norm_eps", 1e-6),
            rope_theta=raw.get("rope_theta", 1_000_000.0),
            max_position_embeddings=raw.get("max_position_embeddings", 32768),
            tie_word_embeddings=raw.get("tie_word_embeddings", True),
            attn_bias=raw.get("attention_bias", raw.get("model_type", "") != "mistral"),
        )

    @property
    def group(self) -> int:
        return self.num_attention_heads // self.num_key_value_heads


# Architectures of the benchmark workloads (random-initialised weights).
PRESETS: dict[str, ModelConfig] = {
    "qwen2.5-0.5b": ModelConfig(),
    "mistral-7b": ModelConfig(hidden_size=4096, num_attention_heads=32, num_key_value_heads=8, head_dim=128,
                              num_hidden_layers=32, intermediate_size=14336, vocab_size=32768,
                              rms_norm_eps=1e-5, rope_theta=1_000_000.0, tie_word_embeddings=False,
                              attn_bias=False),
    "qwen2.5-7b": ModelConfig(hidden_size=3584, num_attention_heads=28, num_key_value_heads=4, head_dim=128,
                              num_hidden_layers=28, intermediate_size=18944, vocab_size=152064,
                              tie_word_embeddings=False, attn_bias=True),
    "qwen2.5-72b": ModelConfig(hidden_size=8192, num_attention_heads=64, num_key_value_heads=8, head_dim=128,
                               num_hidden_layers=80, intermediate_size=29568, vocab_size=152064,
                               tie_word_embeddings=False, attn_bias=True),
}


def precompute_rope(head_dim: int, max_len: int, theta: float, device, dtype) -> tuple[torch.Tensor, torch.Tensor]:
    """cos / sin tables [max_len, head_dim] (model.py:79-89), cast to ``dtype``."""
    inv_freq = 1.0 / (theta ** (torch.arange(0, head_dim, 2, device=device).float() / head_dim))
    t = torch.arange(max_len, device=device, dtype=torch.float32)
    freqs = torch.outer(t, inv_freq)
    emb = torch.cat([freqs, freqs], dim=-1)
    return emb.cos().to(dtype), emb.sin().to(dtype)


def apply_rope(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """Rotate-half RoPE (model.py:92-107); x [T, H, D], cos/sin [T, D]."""
    half = x.shape[-1] // 2
    rotated = torch.cat((-x[..., half:], x[..., :half]), dim=-1)
    return x * cos.unsqueeze(1) + rotated * sin.unsqueeze(1)


class Layer:
    def __init__(self, cfg: ModelConfig, device, dtype, gen: torch.Generator):
        h, d = cfg.hidden_size, cfg.head_dim
        nq, nkv = cfg.num_attention_heads, cfg.num_key_value_heads
        std = 0.02

        def w(*shape):
            return (torch.randn(*shape, device=device, dtype=torch.float32, generator=gen) * std).to(dtype)

        self.in_norm = torch.ones(h, device=device, dtype=dtype)
        self.post_norm = torch.ones(h, device=device, dtype=dtype)
        self.w_qkv = w((nq + 2 * nkv) * d, h)
        self.b_qkv = w((nq + 2 * nkv) * d) if cfg.attn_bias else None
        self.w_o = w(h, nq * d)
        self.w_gate_up = w(2 * cfg.intermediate_size, h)
        self.w_down = w(h, cfg.intermediate_size)
        self.adapters: dict[str, Adapters] = {}


# Schedulers with captured graphs, which hold the addresses of their model's weights.
capturers: weakref.WeakSet = weakref.WeakSet()


def _project(h: torch.Tensor | MXFP8, w: torch.Tensor | MXFP4 | MXFP8, bias: torch.Tensor | None = None) -> torch.Tensor:
    if isinstance(w, MXFP8):
        return linear_mxfp8(h if isinstance(h, MXFP8) else quantize_mxfp8(h), w, bias)
    return linear_mxfp4(h, w, bias) if isinstance(w, MXFP4) else linear(h, w, bias)


# The projections that may have adapters, and the pieces of their outputs, by the names of checkpoints.
ADAPTED = {"w_qkv": ("self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj"), "w_o": ("self_attn.o_proj",),
           "w_gate_up": ("mlp.gate_proj", "mlp.up_proj"), "w_down": ("mlp.down_proj",)}


@dataclasses.dataclass
class AttentionBackend:
    """What the attention layers need for one forward (scheduler.py:229-259).

    ``wrapper`` is a planned decode or prefill wrapper; ``kv_indices`` /
    ``kv_indptr`` / ``kv_last_page_len`` are the CSR page table;
    ``batch_indices`` / ``positions`` place each new token's K/V.
    ``append_indptr`` is carried for interface parity (unused, as in the
    reference).
    """

    paged_kv_cache: object
    wrapper: object
    mode: str
    kv_page_indptr: torch.Tensor
    kv_page_indices: torch.Tensor
    kv_last_page_len: torch.Tensor
    append_indptr: torch.Tensor | None
    batch_indices: torch.Tensor
    positions: torch.Tensor
    _layer_idx: int = 0
    # an ``adapters.AdapterPlan`` of the forward's rows; None: no row has an adapter
    adapter_plan: object | None = None

    def next_layer(self) -> int:
        idx = self._layer_idx
        self._layer_idx += 1
        return idx


class Model:
    def __init__(self, cfg: ModelConfig, device, dtype=torch.bfloat16, seed: int = 0, max_positions: int | None = None,
                 fused_rope: bool = True, fused_dense: bool = True, fused_decode: bool = True):
        self.cfg = cfg
        self.fused_rope = fused_rope
        self.fused_decode = fused_decode
        self.fused_dense = fused_dense
        self.device = torch.device(device)
        self.dtype = dtype
        gen = torch.Generator(device=self.device).manual_seed(seed)
        self.embed = (torch.randn(cfg.vocab_size, cfg.hidden_size, device=self.device, generator=gen) * 0.02).to(dtype)
        self.layers = [Layer(cfg, self.device, dtype, gen) for _ in range(cfg.num_hidden_layers)]
        self.norm = torch.ones(cfg.hidden_size, device=self.device, dtype=dtype)
        self.lm_head = self.embed if cfg.tie_word_embeddings else \
            (torch.randn(cfg.vocab_size, cfg.hidden_size, device=self.device, generator=gen) * 0.02).to(dtype)
        n = max_positions or cfg.max_position_embeddings
        self.cos, self.sin = precompute_rope(cfg.head_dim, n, cfg.rope_theta, self.device, dtype)

    def weight_bytes(self) -> int:
        """Of everything that a forward may read, the adapters' room included."""
        t = self.embed.numel() + self.norm.numel()
        if self.lm_head is not self.embed:
            t += self.lm_head.numel()
        t *= self.embed.element_size()
        for L in self.layers:
            for x in (L.in_norm, L.post_norm, L.w_qkv, L.b_qkv, L.w_o, L.w_gate_up, L.w_down):
                if x is not None:
                    t += x.nbytes
            t += sum(a.nbytes for a in L.adapters.values())
        return t

    def quantize_weights(self, weight_format: str = "mxfp4") -> None:
        """The layers' projections in microscaled floats of 4 bits ("mxfp4", 0.53 bytes per weight) or
        8 ("mxfp8", 1.03) from here on; embedding, LM head, norms and biases stay in bf16.  After the
        weights are loaded and before a scheduler captures its graphs, which read the
        weights of their time.  Weights that have no such form leave the model as it was."""
        if weight_format not in ("mxfp4", "mxfp8"):
            raise ValueError(f"weight_format {weight_format!r}: mxfp4 or mxfp8")
        made, quantize = (MXFP4, quantize_mxfp4) if weight_format == "mxfp4" else (MXFP8, quantize_mxfp8)
        bits = weight_format[-1]
        if not self.fused_dense:
            raise ValueError(f"{bits}-bit weights need fused_dense")
        weights = [(L, name) for L in self.layers for name in ADAPTED if not isinstance(getattr(L, name), made)]
        if weights and any(s.model is self for s in capturers):
            gc.collect()  # (one that nobody holds any more may be part of a cycle)
            if any(s.model is self for s in capturers):
                raise RuntimeError("a scheduler's captured graphs read the weights: quantize_weights() comes before it")
        for L, name in weights:
            w = getattr(L, name)
            if not isinstance(w, torch.Tensor):
                raise ValueError(f"{name} is held in another microscaled format: weights are quantised from bf16")
            if not w.is_cuda or w.dtype != torch.bfloat16 or w.shape[1] % BLOCK:
                raise ValueError(f"{bits}-bit weights are made of bf16 on a GPU with columns in blocks of {BLOCK}; {name} is "
                                 f"{tuple(w.shape)} {w.dtype} on {w.device}")
        for L, name in weights:  # (one by one: both forms of all weights need not fit together)
            setattr(L, name, quantize(getattr(L, name)))

    # ------------------------------------------------------------------ adapters
    @property
    def adapter_slots(self) -> int:
        """How many adapters there is room for."""
        return next((a.slots for L in self.layers for a in L.adapters.values()), 0)

    def enable_adapters(self, slots: int, rank: int, projections=tuple(ADAPTED)) -> None:
        """Room for ``slots`` adapters of up to ``rank`` beside the layers' projections (any of ADAPTED's
        names), which add nothing until ``weights.load_adapter`` or ``Adapters.set`` fills them.  Before a
        scheduler of this model is made."""
        if not self.fused_dense:
            raise ValueError("adapters need fused_dense")
        unknown = set(projections) - set(ADAPTED)
        if unknown or not projections:
            raise ValueError(f"projections {sorted(unknown)}: any of {sorted(ADAPTED)}")
        if self.adapter_slots:
            raise ValueError("the model has adapters already")
        cfg = self.cfg
        q, kv = cfg.num_attention_heads * cfg.head_dim, cfg.num_key_value_heads * cfg.head_dim
        h, inter = cfg.hidden_size, cfg.intermediate_size
        shapes = {"w_qkv": (h, [q, kv, kv]), "w_o": (q, [h]), "w_gate_up": (h, [inter, inter]), "w_down": (inter, [h])}
        made = [{name: Adapters.empty(slots, *shapes[name], rank, self.device) for name in projections} for _ in self.layers]
        for L, adapters in zip(self.layers, made):
            L.adapters = adapters

    # ------------------------------------------------------------------ forward
    def forward(self, input_ids: torch.Tensor, positions: torch.Tensor, backend: AttentionBackend,
                last_rows: torch.Tensor | None = None) -> torch.Tensor:
        """input_ids / positions: [T] (one row per new token).

        Decode: T = batch, returns logits [T, V].  Prefill: T = sum of prompt
        lengths, returns logits [len(last_rows), V] for the rows given.
        """
        cfg = self.cfg
        nq, nkv, d = cfg.num_attention_heads, cfg.num_key_value_heads, cfg.head_dim
        x = F.embedding(input_ids, self.embed)
        fused = self.fused_rope
        if fused:
            rope_pos = positions if positions.dtype == torch.int32 else positions.to(torch.int32)
        else:
            cos = self.cos.index_select(0, positions)
            sin = self.sin.index_select(0, positions)
        t = input_ids.shape[0]
        backend._layer_idx = 0
        eps = cfg.rms_norm_eps
        dense = self.fused_dense
        project = _project if dense else F.linear
        plan = backend.adapter_plan
        if plan is not None and not dense:
            raise ValueError("adapters need fused_dense")

        def adapted(y, h, L, name):  # y, with what the rows' adapters add to it
            adapters = L.adapters.get(name) if plan is not None else None
            return y if adapters is None else add_adapters(y, h, adapters, plan)

        def norm(x, delta, weight, w):  # the norm that w's projection reads
            if isinstance(w, MXFP8):
                return add_rms_norm_mxfp8(x, delta, weight, eps)
            return add_rms_norm(x, delta, weight, eps, write_x=delta is not None)

        if dense:
            h = norm(x, None, self.layers[0].in_norm, self.layers[0].w_qkv)
        for li, L in enumerate(self.layers):
            layer_idx = backend.next_layer()
            if not dense:
                h = F.rms_norm(x, (cfg.hidden_size,), L.in_norm, eps)
            qkv = adapted(project(h, L.w_qkv, L.b_qkv), h, L, "w_qkv")
            kv_data = backend.paged_kv_cache.kv_data[layer_idx]
            if fused and backend.mode == "decode" and self.fused_decode:
                # RoPE, append and attention in one launch (one new token per
                # request, at its last position)
                o = backend.wrapper.run_rope_append(qkv, self.cos, self.sin, kv_data)
            elif fused:
                # q rotated in place in qkv's q columns; k rotated and v appended
                q = rope_append_paged_kv_cache(qkv, nq, nkv, rope_pos, self.cos, self.sin, backend.batch_indices,
                                               backend.positions, kv_data, backend.kv_page_indices,
                                               backend.kv_page_indptr, backend.kv_last_page_len)
            else:
                q = apply_rope(qkv[:, : nq * d].view(t, nq, d), cos, sin)
                k = apply_rope(qkv[:, nq * d: (nq + nkv) * d].view(t, nkv, d), cos, sin)
                v = qkv[:, (nq + nkv) * d:].view(t, nkv, d)
                append_paged_kv_cache(k, v, backend.batch_indices, backend.positions, kv_data,
                                      backend.kv_page_indices, backend.kv_page_indptr, backend.kv_last_page_len)
            if not (fused and backend.mode == "decode" and self.fused_decode):
                o = backend.wrapper.run(q, kv_data)
            if not dense:
                x = x + F.linear(o.view(t, nq * d), L.w_o)
                h = F.rms_norm(x, (cfg.hidden_size,), L.post_norm, eps)
                gu = F.linear(h, L.w_gate_up)
                g, u = gu.chunk(2, dim=-1)
                x = x + F.linear(F.silu(g) * u, L.w_down)
                continue
            # x += o W_o; h = rms(x); x += down(silu(g) * u); h = next layer's rms(x)
            o = o.view(t, nq * d)
            if isinstance(L.w_o, MXFP8):
                o = quantize_mxfp8(o)
            h = norm(x, adapted(project(o, L.w_o), o, L, "w_o"), L.post_norm, L.w_gate_up)
            if plan is not None and "w_gate_up" in L.adapters:
                # (rows without an adapter get the bits of the forms below, whatever rows stand beside them)
                sums = gate_up_mxfp8 if isinstance(L.w_gate_up, MXFP8) else gate_up_mxfp4 if isinstance(L.w_gate_up, MXFP4) else linear
                act = add_adapters_silu(sums(h, L.w_gate_up), h, L.adapters["w_gate_up"], plan,
                                        quantize=isinstance(L.w_gate_up, MXFP8), stepwise=sums is linear)
            elif isinstance(L.w_gate_up, MXFP8):
                act = linear_silu_mxfp8(h, L.w_gate_up, quantize=True)
            else:
                act = (linear_silu_mxfp4 if isinstance(L.w_gate_up, MXFP4) else linear_silu)(h, L.w_gate_up)
            down = adapted(project(act, L.w_down), act, L, "w_down")
            if li + 1 < len(self.layers):
                nxt = self.layers[li + 1]
                h = norm(x, down, nxt.in_norm, nxt.w_qkv)
            elif last_rows is None:
                h = add_rms_norm(x, down, self.norm, eps)
            else:
                add_rms_norm(x, down, None, eps, norm=False)
                h = add_rms_norm(x.index_select(0, last_rows), None, self.norm, eps, write_x=False)
        if not dense:
            if last_rows is not None:
                x = x.index_select(0, last_rows)
            h = F.rms_norm(x, (cfg.hidden_size,), self.norm, eps)
        return project(h, self.lm_head)


def kv_pool_bytes_per_page(cfg: ModelConfig, page_size: int = 16) -> int:
    return 2 * page_size * cfg.num_key_value_heads * cfg.head_dim * 2 * cfg.num_hidden_layers


def default_pages(cfg: ModelConfig, max_batch: int, max_seq_len: int, page_size: int = 16) -> int:
    return max_batch * math.ceil(max_seq_len / page_size)
