"""Workloads of the operators around a decode step's attention: microscaled 4-bit
quantisation, the projections it feeds, the norms before and after a block, and the
filtered draw from given random numbers.

``run`` computes each in elementary torch operations, or, where ``own`` is true, by
the calls that a user makes of this framework.  Widths are those of the model presets
(projections of Mistral-7B and Qwen2.5-0.5B / 7B / 72B), rows those of decode batches
and of the benchmark's prompts.

Kinds of case:

  quantize  rows of activations into microscaled 4-bit floating point and back
  linear    a projection whose weight is held in 4 bits; the activations are bf16, or
            (``acts`` "mxfp4") are quantised within the call; with ``silu`` the fused
            gate and up projection followed by silu(gate) * up
  norms     norm of a block's output, gate, residual scale, sum, norm before the next block
  sample    one draw per row with temperature, top-k, top-p and min-p
"""

from __future__ import annotations

import math
import random

import torch

own = False

BLOCK = 32
EPS = 1e-6
GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]  # magnitudes of the eight codes

# (k, n, gated) of the presets' projections: qkv, o, gate and up (n: outputs of the gated product), down
PROJECTIONS = [
    (896, 1152, False), (896, 896, False), (896, 4864, True), (4864, 896, False),
    (4096, 6144, False), (4096, 4096, False), (4096, 14336, True), (14336, 4096, False),
    (3584, 4608, False), (3584, 3584, False), (3584, 18944, True), (18944, 3584, False),
    (8192, 10240, False), (8192, 8192, False), (8192, 29568, True), (29568, 8192, False),
]
VOCABS = [32768, 151936, 152064]
GATES = ["none", "channel", "token", "full"]


# ------------------------------------------------------------------ the cases
def _linear(rows, k, n, acts="bf16", silu=False, bias=False):
    return {"kind": "linear", "rows": rows, "k": k, "n": n, "acts": acts, "silu": silu, "bias": bias}


def listed():
    return [
        # a small decode batch's activations, Qwen2.5-0.5B width: latency
        {"name": "quantize_decode_rows", "kind": "quantize", "rows": 8, "cols": 896},
        # the activations of the benchmark's 32 prompts at Mistral-7B's width
        {"name": "quantize_prompt_rows", "kind": "quantize", "rows": 18240, "cols": 4096},
        # one token through Qwen2.5-0.5B's gate and up projection
        {"name": "linear_one_token", **_linear(1, 896, 4864, silu=True)},
        # the benchmark's decode batch through Mistral-7B's gate and up projection
        {"name": "linear_batch_32", **_linear(32, 4096, 14336, silu=True)},
        # a short prompt of odd length through Qwen2.5-7B's down projection
        {"name": "linear_short_prompt", **_linear(77, 18944, 3584)},
        # prompts admitted together through Mistral-7B's fused q, k and v, 4-bit weights only
        {"name": "linear_prompt_rows", **_linear(4105, 4096, 6144)},
        # a wide decode batch, both sides in 4 bits, Qwen2.5-72B's fused q, k and v with their bias
        {"name": "product_batch_48", **_linear(48, 8192, 10240, acts="mxfp4", bias=True)},
        # eight long prompts, both sides in 4 bits, the same projection
        {"name": "product_prompt_rows", **_linear(8201, 8192, 10240, acts="mxfp4", bias=True)},
        # a decode batch between two blocks of Qwen2.5-72B's width
        {"name": "norms_batch_32", "kind": "norms", "rows": 32, "hidden": 8192, "gate": "none"},
        # the benchmark's prompt rows with a gate of one value per channel
        {"name": "norms_prompt_rows", "kind": "norms", "rows": 18240, "hidden": 4096, "gate": "channel"},
        # the draw of one stream, Mistral-7B's vocabulary
        {"name": "sample_one_stream", "kind": "sample", "batch": 1, "vocab": 32768},
        # the draw of a 48-request step at the Qwen vocabulary
        {"name": "sample_batch_48", "kind": "sample", "batch": 48, "vocab": 152064},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    """One more case: any operator, any size of the served range."""
    kind = rng.choice(["quantize", "linear", "linear", "linear", "linear", "norms", "sample", "sample"])
    if kind == "quantize":
        cols = BLOCK * _log_int(rng, 1, 29568 // BLOCK)
        return {"kind": kind, "rows": _log_int(rng, 1, min(18240, 18240 * 4096 // cols)), "cols": cols}
    if kind == "norms":
        hidden = 8 * _log_int(rng, 8, 16384 // 8)
        return {"kind": kind, "rows": _log_int(rng, 1, min(18240, 18240 * 4096 // hidden)), "hidden": hidden,
                "gate": rng.choice(GATES)}
    if kind == "sample":
        vocab = rng.choice(VOCABS) - rng.choice([0, 0, 7])
        if rng.random() < 0.25:
            vocab = _log_int(rng, 100, 30000)
        return {"kind": kind, "batch": _log_int(rng, 1, 64 if vocab < 100000 else 48), "vocab": vocab}
    k, n, silu = rng.choice(PROJECTIONS)
    if rng.random() < 0.3:  # widths that fill no whole tile
        k, n = k - BLOCK * rng.randrange(4), n - rng.randrange(16)
    wide = n * (2 if silu else 1) * k
    rows = _log_int(rng, 1, max(1, min(8201, 8201 * 8192 * 10240 // wide)))
    return _linear(rows, k, n, rng.choice(["bf16", "bf16", "mxfp4"]), silu, rng.random() < 0.3 and not silu)


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _activations(rows, cols, gen):
    """Rows after a norm: unit scale with a few channels that stand out, as in trained models."""
    x = torch.randn(rows, cols, device="cuda", generator=gen)
    channel = torch.randn(cols, device="cuda", generator=gen).mul_(0.3).exp_()
    loud = torch.rand(cols, device="cuda", generator=gen) < 0.004
    return (x * torch.where(loud, 12.0 * channel, channel)).to(torch.bfloat16)


def _weight_parts(n, k, gen):
    """A weight as a checkpoint holds it: scale bytes [n, k / 32] and codes, two to a byte, [n, k / 2]
    (the lower half first), for normal values of a spread that differs from row to row."""
    spread = torch.randn(n, 1, device="cuda", generator=gen).mul_(0.2).exp_().mul_(0.02)
    w = torch.randn(n, k, device="cuda", generator=gen).mul_(spread).view(n, k // BLOCK, BLOCK)
    e = torch.frexp(w.abs().amax(-1))[1] - 3  # amax = m 2^x with m in [1/2, 1): floor(log2 amax) - 2
    w = torch.ldexp(w, -e[..., None])
    code = _codes(w).view(n, k // 2, 2)
    return (e + 127).to(torch.uint8), code[..., 0] | (code[..., 1] << 4)


def _inputs(case, seed):
    """The inputs of a case, alike for both forms and for ``exact``."""
    gen, kind = _gen(seed), case["kind"]
    if kind == "quantize":
        return {"x": _activations(case["rows"], case["cols"], gen)}
    if kind == "linear":
        n = case["n"] * (2 if case["silu"] else 1)
        scales, codes = _weight_parts(n, case["k"], gen)
        x = {"x": _activations(case["rows"], case["k"], gen), "scales": scales, "codes": codes, "bias": None}
        if case["bias"]:
            x["bias"] = torch.randn(n, device="cuda", generator=gen).to(torch.bfloat16)
        return x
    if kind == "norms":
        rows, hidden = case["rows"], case["hidden"]

        def randn(*shape):
            return torch.randn(*shape, device="cuda", dtype=torch.bfloat16, generator=gen)

        gate = {"none": None, "channel": (hidden,), "token": (rows, 1), "full": (rows, hidden)}[case["gate"]]
        return {"x": 3.0 * randn(rows, hidden), "y": randn(rows, hidden), "post": 1 + 0.1 * randn(hidden),
                "pre": 1 + 0.1 * randn(hidden), "gate": None if gate is None else torch.sigmoid(randn(*gate))}
    n = case["batch"]
    logits = torch.randn(n, case["vocab"], device="cuda", generator=gen).mul_(3.0).to(torch.bfloat16)
    row = torch.arange(n, device="cuda")
    # requests of a server: greedy, plain temperature, top-k, top-p, min-p, and all three together
    return {
        "logits": logits, "u": torch.rand(n, device="cuda", generator=gen),
        "temperature": torch.where(row % 8 == 3, 0.0, 0.6 + 0.1 * (row % 7).float()),
        "top_k": torch.where((row % 4 == 0) | (row % 8 == 5), 20 + 30 * (row % 5), 0).to(torch.int32),
        "top_p": torch.where((row % 4 == 1) | (row % 8 == 4), 0.8 + 0.03 * (row % 6).float(), 1.0),
        "min_p": torch.where((row % 4 == 2) | (row % 8 == 5), 0.02 + 0.02 * (row % 3).float(), 0.0),
    }


def prepare(case, seed):
    x = _inputs(case, seed)
    state = {"case": case, **x}
    if case["kind"] == "linear":
        state["values"] = _values(x["codes"], x["scales"]).to(torch.bfloat16)  # exact: three bits and a power of two
    if own:  # the weight's and the sampler's handles, which a program keeps
        import __graft_entry__

        __graft_entry__.load_package()
        if case["kind"] == "linear":
            from minimal_inference_amd.mxfp4 import MXFP4

            state["weight"] = MXFP4.from_codes(x["codes"].to(torch.uint8), x["scales"])
        if case["kind"] == "sample":
            from minimal_inference_amd.sampling import Sampler

            s = state["sampler"] = Sampler(torch.device("cuda"), case["batch"], vocab=case["vocab"])
            s.set_params(x["temperature"], x["top_p"], top_k=x["top_k"], min_p=x["min_p"])
    return state


# ------------------------------------------------------------------ plain forms
def _codes(v):
    """Codes of scaled values: the nearest of the grid, ties to the even code, 6 at most."""
    a = v.abs()
    mag = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    return mag + 8 * torch.signbit(v)


def _values(codes, scales):
    """What packed codes and scale bytes stand for, in 32 bits."""
    n, half = codes.shape
    code = torch.stack((codes & 15, codes >> 4), -1).view(n, 2 * half // BLOCK, BLOCK).int()
    grid = torch.tensor(GRID, device=codes.device)
    value = torch.where(code < 8, grid[code & 7], -grid[code & 7])
    return torch.ldexp(value, (scales.int() - 127)[..., None]).view(n, 2 * half)


def _quantized(x):
    """The values that rows hold after quantisation, in 32 bits."""
    rows, cols = x.shape
    v = x.float().view(rows, cols // BLOCK, BLOCK)
    amax = v.abs().amax(-1)
    e = torch.where(amax > 0, torch.frexp(amax)[1] - 3, -127).clamp_(-127, 127)[..., None]
    code = _codes(torch.ldexp(v, -e)).int()
    grid = torch.tensor(GRID, device=x.device)
    value = torch.where(code < 8, grid[code & 7], -grid[code & 7])
    return torch.ldexp(value, e).view(rows, cols)


def _plain_norms(s):
    x, y = s["x"].float(), s["y"].float()
    z = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * s["post"].float()
    if s["gate"] is not None:
        z = z * s["gate"].float()
    x = x + 0.25 * z
    h = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * s["pre"].float()
    return {"x": x.to(torch.bfloat16), "h": h.to(torch.bfloat16)}


def _plain_draw(s):
    """In 64 bits: a draw close to a border between two tokens has to fall on the right side."""
    value, index = torch.sort(s["logits"].double(), dim=-1, descending=True, stable=True)
    t = s["temperature"].double()[:, None]
    greedy = t <= 0
    w = torch.exp((value - value[:, :1]) / torch.where(greedy, 1.0, t))
    rank = torch.arange(w.shape[1], device=w.device)
    top_k, top_p, min_p = s["top_k"][:, None], s["top_p"].double()[:, None], s["min_p"].double()[:, None]
    w = torch.where(((top_k <= 0) | (rank < top_k)) & (w >= min_p), w, 0.0)
    before = torch.cumsum(w, -1) - w
    kept = (top_p >= 1) | (before < top_p * w.sum(-1, keepdim=True)) | (rank == 0)
    weight = torch.zeros_like(w).scatter_(1, index, torch.where(kept, w, 0.0))
    cum = torch.cumsum(weight, -1)
    drawn = (cum > s["u"].double()[:, None] * cum[:, -1:]).to(torch.uint8).argmax(-1)
    return torch.where(greedy[:, 0], index[:, 0], drawn)


def _plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "quantize":
        return _quantized(s["x"]).to(torch.bfloat16)
    if kind == "norms":
        return _plain_norms(s)
    if kind == "sample":
        return _plain_draw(s)
    x = _quantized(s["x"]) if case["acts"] == "mxfp4" else s["x"].float()
    y = x @ s["values"].float().t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if case["silu"]:
        gate, up = y.chunk(2, dim=-1)
        y = gate / (1 + torch.exp(-gate)) * up
    return y.to(torch.bfloat16)


# ------------------------------------------------------------------ run
def run(state):
    if not own:
        return _plain(state)
    case = state["case"]
    kind = case["kind"]
    if kind == "quantize":
        from minimal_inference_amd.mxfp4 import quantize_mxfp4

        return quantize_mxfp4(state["x"]).dequantize()
    if kind == "norms":
        from minimal_inference_amd.dense import post_norm_add_rms_norm

        x = torch.empty_like(state["x"])
        h = post_norm_add_rms_norm(state["x"], state["y"], state["post"], state["pre"], EPS, gate=state["gate"],
                                   scale=0.25, x_out=x)
        return {"x": x, "h": h}
    if kind == "sample":
        return state["sampler"].draw(state["logits"], state["u"])
    from minimal_inference_amd.mxfp4 import linear_mxfp4, linear_silu_mxfp4, quantize_mxfp4

    x = quantize_mxfp4(state["x"]) if case["acts"] == "mxfp4" else state["x"]
    if case["silu"]:
        return linear_silu_mxfp4(x, state["weight"])
    return linear_mxfp4(x, state["weight"], state["bias"])


# ------------------------------------------------------------------ work
def work(case):
    kind = case["kind"]
    if kind == "quantize":
        return {"bytes": 4 * case["rows"] * case["cols"], "flops": 0}
    if kind == "norms":
        rows, hidden = case["rows"], case["hidden"]
        gate = {"none": 0, "channel": hidden, "token": rows, "full": rows * hidden}[case["gate"]]
        return {"bytes": 8 * rows * hidden + 4 * hidden + 2 * gate, "flops": 0}
    if kind == "sample":
        return {"bytes": case["batch"] * (2 * case["vocab"] + 28), "flops": 0}
    rows, k, n = case["rows"], case["k"], case["n"] * (2 if case["silu"] else 1)
    weight = n * k // 2 + n * k // BLOCK
    return {"bytes": weight + 2 * rows * k + 2 * rows * case["n"] + (2 * n if case["bias"] else 0),
            "flops": 2 * rows * n * k}


# ------------------------------------------------------------------ exact
def _exact_quantized(x):
    """Each value replaced by the nearest that its block can hold, in 64 bits: the block's unit is
    2^(floor(log2 amax) - 2), and of two as near the one whose place in the grid is even."""
    rows, cols = x.shape
    v = x.double().view(rows, cols // BLOCK, BLOCK)
    amax = v.abs().amax(-1, keepdim=True)
    bits = amax.view(torch.int64)
    unit = torch.where(amax > 0, ((bits >> 52) - 1023 - 2).clamp(-127, 127), -127).double().exp2()
    a = (v / unit).abs().clamp(max=6.0)
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).double()
    return (torch.round(a / step) * step * unit * torch.sign(v)).view(rows, cols)  # round: halves to even


def exact(case, seed):
    kind = case["kind"]
    if kind == "sample":
        return None  # token ids: no computed number
    s = _inputs(case, seed)
    if kind == "quantize":
        return _exact_quantized(s["x"])
    if kind == "norms":
        x, y = s["x"].double(), s["y"].double()
        gate = 1.0 if s["gate"] is None else s["gate"].double()
        x = x + y / (y.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * (s["post"].double() * 0.25) * gate
        return {"x": x, "h": x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * s["pre"].double()}
    x = _exact_quantized(s["x"]) if case["acts"] == "mxfp4" else s["x"].double()
    codes, unit = s["codes"], (s["scales"].double() - 127).exp2()
    table = torch.tensor(GRID + [-v for v in GRID], dtype=torch.float64, device=codes.device)
    w = torch.empty(codes.shape[0], 2 * codes.shape[1], dtype=torch.float64, device=codes.device)
    w[:, 0::2], w[:, 1::2] = table[(codes & 15).long()], table[(codes >> 4).long()]
    w = (w.view(-1, unit.shape[1], BLOCK) * unit[..., None]).view(w.shape)
    y = torch.matmul(x, w.t())
    if s["bias"] is not None:
        y += s["bias"].double()
    if case["silu"]:
        gate, up = y.chunk(2, dim=-1)
        y = gate * torch.sigmoid(gate) * up
    return y
