"""Workloads of the 8-bit side of a block and of the adapters that requests bring along:
the residual sum and norm that leaves microscaled 8-bit rows, the projections over such
rows, and low-rank adapters of many requests beside a shared projection.

``run`` computes each in elementary torch operations, or, where ``own`` is true, by
the calls that a user makes of this framework.  Widths are those of the model presets
(projections of Mistral-7B and Qwen2.5-0.5B / 7B / 72B), rows those of decode batches
and of the benchmark's prompts.

Kinds of case:

  norm     x + delta, its root-mean-square norm, and that in 8 bits: blocks of 32 with a
           power of two each; returns the sum and the values that the blocks stand for
  linear   a projection with both operands in 8 bits; with ``silu`` the fused gate and up
           projection followed by silu(gate) * up
  adapter  y + scale B (A x) with the row's own adapter, of several requests at once; the
           outputs are one piece (o, down) or several with factors of their own (q, k, v);
           x is bf16 or (``acts`` "mxfp8") 8-bit rows; an eighth of the requests has none
"""

from __future__ import annotations

import math

import torch

own = False

BLOCK = 32
EPS = 1e-6
LARGEST = 448.0  # of e4m3

# (k, n, gated) of the presets' projections: qkv, o, gate and up (n: outputs of the gated product), down
PROJECTIONS = [
    (896, 1152, False), (896, 896, False), (896, 4864, True), (4864, 896, False),
    (4096, 6144, False), (4096, 4096, False), (4096, 14336, True), (14336, 4096, False),
    (3584, 4608, False), (3584, 3584, False), (3584, 18944, True), (18944, 3584, False),
    (8192, 10240, False), (8192, 8192, False), (8192, 29568, True), (29568, 8192, False),
]
# (k, outputs of the pieces) of the same projections with adapters
ADAPTED = [
    (896, "896,128,128"), (896, "896"), (896, "4864,4864"), (4864, "896"),
    (4096, "4096,1024,1024"), (4096, "4096"), (4096, "14336,14336"), (14336, "4096"),
    (3584, "3584,512,512"), (3584, "3584"), (3584, "18944,18944"), (18944, "3584"),
    (8192, "8192,1024,1024"), (8192, "8192"), (29568, "8192"),
]


# ------------------------------------------------------------------ the cases
def _norm(rows, hidden, delta=True):
    return {"kind": "norm", "rows": rows, "hidden": hidden, "delta": delta}


def _linear(rows, k, n, silu=False, bias=False):
    return {"kind": "linear", "rows": rows, "k": k, "n": n, "silu": silu, "bias": bias}


def _adapter(rows, requests, k, pieces, rank, slots, acts="bf16"):
    return {"kind": "adapter", "rows": rows, "requests": requests, "k": k, "pieces": pieces, "rank": rank,
            "slots": slots, "acts": acts}


def listed():
    return [
        # one token of Qwen2.5-0.5B: latency
        {"name": "norm_one_token", **_norm(1, 896)},
        # a 48-request decode step of Qwen2.5-72B
        {"name": "norm_batch_48", **_norm(48, 8192)},
        # the benchmark's 32 prompts at Mistral-7B's width
        {"name": "norm_prompt_rows", **_norm(18240, 4096)},
        # one token through Mistral-7B's gate and up projection
        {"name": "linear_one_token", **_linear(1, 4096, 14336, silu=True)},
        # the benchmark's decode batch through Mistral-7B's fused q, k and v
        {"name": "linear_batch_32", **_linear(32, 4096, 6144)},
        # a short prompt of odd length through Qwen2.5-7B's down projection
        {"name": "linear_short_prompt", **_linear(77, 18944, 3584)},
        # prompts admitted together through Mistral-7B's gate and up projection
        {"name": "linear_prompt_rows", **_linear(2057, 4096, 14336, silu=True)},
        # eight long prompts through Qwen2.5-72B's fused q, k and v with their bias
        {"name": "linear_long_prompts", **_linear(8201, 8192, 10240, bias=True)},
        # one stream with an adapter on Mistral-7B's output projection: latency
        {"name": "adapter_one_token", **_adapter(1, 1, 4096, "4096", 16, 4)},
        # a 48-request decode step of Qwen2.5-7B, 24 adapters on q, k and v
        {"name": "adapter_batch_48", **_adapter(48, 48, 3584, "3584,512,512", 16, 24)},
        # a decode step in 8 bits with adapters of a large rank on Mistral-7B's down projection
        {"name": "adapter_batch_32_8bit", **_adapter(32, 32, 14336, "4096", 64, 8, acts="mxfp8")},
        # the benchmark's 32 prompts, 8 adapters on Mistral-7B's q, k and v
        {"name": "adapter_prompt_rows", **_adapter(18240, 32, 4096, "4096,1024,1024", 16, 8)},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    """One more case: any operator, any size of the served range."""
    kind = rng.choice(["norm", "linear", "linear", "linear", "adapter", "adapter"])
    if kind == "norm":
        hidden = BLOCK * _log_int(rng, 2, 16384 // BLOCK)
        return _norm(_log_int(rng, 1, min(18240, 18240 * 4096 // hidden)), hidden, rng.random() < 0.75)
    if kind == "linear":
        k, n, silu = rng.choice(PROJECTIONS)
        if rng.random() < 0.3:  # widths that fill no whole tile
            k, n = k - BLOCK * rng.randrange(4), n - rng.randrange(16)
        wide = n * (2 if silu else 1) * k
        rows = _log_int(rng, 1, max(1, min(8201, 8201 * 8192 * 10240 // wide)))
        return _linear(rows, k, n, silu, rng.random() < 0.3 and not silu)
    k, pieces = rng.choice(ADAPTED)
    wide = k + 2 * sum(int(p) for p in pieces.split(","))
    rows = _log_int(rng, 1, min(18240, 18240 * 16384 // wide))
    requests = rows if rows <= 64 else rng.randint(1, 64)
    slots = _log_int(rng, 1, 32)
    return _adapter(rows, requests, k, pieces, rng.choice([8, 16, 16, 24, 32, 64]), slots, rng.choice(["bf16", "mxfp8"]))


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _activations(rows, cols, gen):
    """Rows after a norm: unit scale with a few channels that stand out, as in trained models."""
    x = torch.randn(rows, cols, device="cuda", generator=gen)
    channel = torch.randn(cols, device="cuda", generator=gen).mul_(0.3).exp_()
    loud = torch.rand(cols, device="cuda", generator=gen) < 0.004
    return x.mul_(torch.where(loud, 12.0 * channel, channel))


def _quantized(v):
    """Codes (e4m3, [rows, cols]) and scale bytes ([rows, cols / 32]) of fp32 rows: a block's
    power of two is the least that keeps all of it within 448."""
    rows, cols = v.shape
    v = v.view(rows, cols // BLOCK, BLOCK)
    m, e = torch.frexp(v.abs().amax(-1))  # amax = m 2^e with m in [1/2, 1), 448 = 7/8 2^9
    e = torch.where(m > 0, e - 9 + (m > LARGEST / 512).to(e.dtype), -127).clamp_(-127, 127)
    codes = torch.ldexp(v, -e[..., None]).to(torch.float8_e4m3fn).view(rows, cols)
    return codes, (e + 127).to(torch.uint8)


def _values(codes, scales):
    """What codes and scale bytes stand for, in 32 bits."""
    rows, cols = codes.shape
    v = codes.float().view(rows, cols // BLOCK, BLOCK)
    return torch.ldexp(v, (scales.int() - 127)[..., None]).view(rows, cols)


def _pieces(case):
    return [int(p) for p in case["pieces"].split(",")]


def _slot_of(request, slots):
    """The adapter of a request, -1 for none."""
    return -1 if request % 8 == 7 else request % slots


def _inputs(case, seed):
    """The inputs of a case, alike for both forms and for ``exact``."""
    gen, kind, rows = _gen(seed), case["kind"], case["rows"]

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    if kind == "norm":
        hidden = case["hidden"]
        return {"x": (3.0 * _activations(rows, hidden, gen)).to(torch.bfloat16),
                "delta": randn(rows, hidden).to(torch.bfloat16) if case["delta"] else None,
                "weight": (1 + 0.1 * randn(hidden)).to(torch.bfloat16)}
    if kind == "linear":
        n, k = case["n"] * (2 if case["silu"] else 1), case["k"]
        w = randn(n, k).mul_(randn(n, 1).mul_(0.2).exp_().mul_(0.7 * k ** -0.5))
        w_codes, w_scales = _quantized(w)
        codes, scales = _quantized(_activations(rows, k, gen))
        return {"codes": codes, "scales": scales, "w_codes": w_codes, "w_scales": w_scales,
                "bias": randn(n).to(torch.bfloat16) if case["bias"] else None}
    k, rank, slots, pieces = case["k"], case["rank"], case["slots"], _pieces(case)
    n = sum(pieces)
    x = _activations(rows, k, gen)
    s = {"y": randn(rows, n).to(torch.bfloat16),
         # trained factors: A near its uniform start of 1 / sqrt(k), B grown to a tenth of the projection
         "a": (randn(slots, len(pieces) * rank, k) * k ** -0.5).to(torch.bfloat16),
         "b": (randn(slots, n, rank) * (0.2 * rank ** -0.5)).to(torch.bfloat16),
         "scale": torch.where(torch.arange(slots, device="cuda") % 2 == 0, 2.0, 0.5)}
    request = torch.arange(rows, device="cuda") * case["requests"] // rows
    s["slot"] = torch.where(request % 8 == 7, -1, request % slots).to(torch.int32)
    if case["acts"] == "mxfp8":
        s["codes"], s["scales"] = _quantized(x)
    else:
        s["x"] = x.to(torch.bfloat16)
    return s


def prepare(case, seed):
    state = {"case": case, **_inputs(case, seed)}
    if own:  # the matrices, the adapters and the batch's plan, which a program keeps
        import __graft_entry__

        __graft_entry__.load_package()
        from minimal_inference_amd.mxfp8 import MXFP8

        if "codes" in state:
            state["rows8"] = MXFP8.from_codes(state["codes"], state["scales"])
        if case["kind"] == "linear":
            state["weight8"] = MXFP8.from_codes(state["w_codes"], state["w_scales"])
        if case["kind"] == "adapter":
            from minimal_inference_amd.adapters import AdapterPlan, Adapters

            state["adapters"] = Adapters(state["a"], state["b"], state["scale"], _pieces(case))
            state["plan"] = AdapterPlan(case["rows"], case["slots"], torch.device("cuda"))
            state["plan"].plan(state["slot"])
    return state


# ------------------------------------------------------------------ plain forms
def _plain_norm(s):
    x = s["x"] if s["delta"] is None else (s["x"].float() + s["delta"].float()).to(torch.bfloat16)
    v = x.float()
    h = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS) * s["weight"].float()
    return {"x": None if s["delta"] is None else x, "h": _values(*_quantized(h)).to(torch.bfloat16)}


def _plain_linear(s):
    y = _values(s["codes"], s["scales"]) @ _values(s["w_codes"], s["w_scales"]).t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if s["case"]["silu"]:
        gate, up = y.chunk(2, dim=-1)
        y = gate / (1 + torch.exp(-gate)) * up
    return y.to(torch.bfloat16)


def _plain_adapter(s):
    """Every row times every adapter's A, the other adapters' parts set to zero, times all B side by side."""
    case = s["case"]
    rows, rank, slots, pieces = case["rows"], case["rank"], case["slots"], _pieces(case)
    x = s["x"].float() if case["acts"] == "bf16" else _values(s["codes"], s["scales"])
    v = (x @ s["a"].float().view(-1, case["k"]).t()).view(rows, slots, len(pieces), rank)
    mine = s["slot"][:, None] == torch.arange(slots, device="cuda")
    v = torch.where(mine[..., None, None], v * s["scale"][:, None, None], 0.0)
    b = torch.split(s["b"].float(), pieces, dim=1)  # per piece [slots, n, rank]
    z = [v[:, :, i].reshape(rows, slots * rank) @ w.transpose(1, 2).reshape(slots * rank, -1) for i, w in enumerate(b)]
    return (s["y"].float() + torch.cat(z, 1)).to(torch.bfloat16)


# ------------------------------------------------------------------ run
def run(state):
    case = state["case"]
    kind = case["kind"]
    if not own:
        return {"norm": _plain_norm, "linear": _plain_linear, "adapter": _plain_adapter}[kind](state)
    if kind == "norm":
        from minimal_inference_amd.mxfp8 import add_rms_norm_mxfp8

        x = None if state["delta"] is None else torch.empty_like(state["x"])
        h = add_rms_norm_mxfp8(state["x"], state["delta"], state["weight"], EPS, x_out=x)
        return {"x": x, "h": h.dequantize()}
    if kind == "adapter":
        from minimal_inference_amd.adapters import add_adapters

        x = state["x"] if case["acts"] == "bf16" else state["rows8"]
        return add_adapters(state["y"], x, state["adapters"], state["plan"], out=torch.empty_like(state["y"]))
    from minimal_inference_amd.mxfp8 import linear_mxfp8, linear_silu_mxfp8

    if case["silu"]:
        return linear_silu_mxfp8(state["rows8"], state["weight8"])
    return linear_mxfp8(state["rows8"], state["weight8"], state["bias"])


# ------------------------------------------------------------------ work
def work(case):
    kind, rows = case["kind"], case["rows"]
    if kind == "norm":
        hidden = case["hidden"]
        return {"bytes": rows * hidden * (8 if case["delta"] else 4) + 2 * hidden, "flops": 0}
    if kind == "linear":
        k, n = case["k"], case["n"] * (2 if case["silu"] else 1)
        return {"bytes": (n + rows) * (k + k // BLOCK) + 2 * rows * case["n"] + (2 * n if case["bias"] else 0),
                "flops": 2 * rows * n * k}
    k, rank, pieces = case["k"], case["rank"], _pieces(case)
    of = [_slot_of(r, case["slots"]) for r in range(case["requests"])]
    each = 2 * rank * (len(pieces) * k + sum(pieces))  # bytes of an adapter, operations of a row
    share = sum(o >= 0 for o in of) / len(of)
    acts = 2 * k if case["acts"] == "bf16" else k + k // BLOCK
    return {"bytes": round(rows * (acts * share + 4 * sum(pieces) + 4)) + len(set(of) - {-1}) * each,
            "flops": round(rows * share * each)}


# ------------------------------------------------------------------ exact
def _exact_quantized(v):
    """Each value replaced by the nearest that its block can hold, in 64 bits: the block's
    unit is the least power of two of which 448 are no less than its largest magnitude, and of two as near
    the one whose place among the unit's fractions is even."""
    rows, cols = v.shape
    v = v.view(rows, cols // BLOCK, BLOCK)
    amax = v.abs().amax(-1, keepdim=True)
    unit = torch.ceil(torch.log2(amax.clamp(min=2.0 ** -150) / LARGEST)).clamp(-127, 127).exp2()
    unit = torch.where(amax > LARGEST * unit, unit * 2, torch.where(amax <= LARGEST / 2 * unit, unit / 2, unit))
    a = v.abs() / unit.clamp(min=2.0 ** -127)
    step = torch.floor(torch.log2(a.clamp(min=2.0 ** -6))).exp2() / 8
    step = torch.where(a < 8 * step, step / 2, step).clamp(min=2.0 ** -9)
    return (torch.round(a / step) * step * unit.clamp(min=2.0 ** -127) * torch.sign(v)).view(rows, cols)


def _exact_values(codes, scales):
    v = codes.double().view(codes.shape[0], -1, BLOCK) * (scales.double() - 127).exp2()[..., None]
    return v.view(codes.shape)


def exact(case, seed):
    kind = case["kind"]
    s = _inputs(case, seed)
    if kind == "norm":
        x = s["x"].double()
        if s["delta"] is not None:
            x = (x + s["delta"].double()).to(torch.bfloat16).double()
        h = x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * s["weight"].double()
        return {"x": None if s["delta"] is None else x, "h": _exact_quantized(h)}
    if kind == "linear":
        y = torch.matmul(_exact_values(s["codes"], s["scales"]), _exact_values(s["w_codes"], s["w_scales"]).t())
        if s["bias"] is not None:
            y += s["bias"].double()
        if case["silu"]:
            gate, up = y.chunk(2, dim=-1)
            y = (gate * torch.sigmoid(gate)).mul_(up)
        return y
    # adapter by adapter, on the rows that are its own
    x = s["x"].double() if case["acts"] == "bf16" else _exact_values(s["codes"], s["scales"])
    y, pieces, rank = s["y"].double(), _pieces(case), case["rank"]
    for slot in range(case["slots"]):
        mine = (s["slot"] == slot).nonzero()[:, 0]
        v = torch.matmul(x[mine], s["a"][slot].double().t()) * s["scale"][slot].double()
        first = 0
        for i, n in enumerate(pieces):
            z = torch.matmul(v[:, i * rank: (i + 1) * rank], s["b"][slot, first: first + n].double().t())
            y[mine, first: first + n] += z
            first += n
    return y
