"""GPU: a model with 8-bit layers and with adapters, against a restatement in 64 bits; a
scheduler and the server's engine over them; adapters from files.

Bars of logits, as max |engine - restated| / max |restated|. Layers in bf16: both sides round the same
quantities at the same places and differ where a rounding falls on the other side of a border, as the fused
and unfused kernels do: 4e-2 (tests/helpers.py). Layers in 8 bits: rows that differ by d (relative) before
they are rounded to e4m3 (relative step s, 2^-4 to 2^-3, 2^-3.5 in the mean of squares) have codes that differ by
sqrt(d s) in the root mean square, since a value crosses a border with probability d / s and moves by s. From
bf16's d = 2^-9 one rounding makes 1.3e-2 of that and the next 3.4e-2, which is where two
independent roundings end: s sqrt(2 / 12) = 3.6e-2 each. Products keep a relative error and norms too; with twelve
such roundings (four a layer, three layers) that add in squares it is sqrt(12) 3.6e-2 = 0.125, and no residual path is
counted, which only dilutes it. Logits and their differences are sums of many terms alike, so the ratio of the maxima
is that of the root mean squares. A mistake (an adapter on another row, a missing scale) moves them
by a few tenths.
"""

from __future__ import annotations

import json

import pytest
import torch

from oracle import mxfp8 as om8
from tests.helpers import E2E_LOGIT_REL_BOUND

pytestmark = pytest.mark.gpu

BOUND_8_BIT = 0.125

NAMES = ("w_qkv", "w_o", "w_gate_up", "w_down")


def _model(dev, seed=3, bias=True):
    from minimal_inference_amd.model import Model, ModelConfig

    cfg = ModelConfig(hidden_size=256, num_attention_heads=6, num_key_value_heads=2, head_dim=64, num_hidden_layers=3,
                      intermediate_size=672, vocab_size=4096, max_position_embeddings=512, attn_bias=bias)
    return Model(cfg, dev, seed=seed, max_positions=512)


def _fill(model, slot, seed, names=NAMES, size=1.0):
    """A random adapter of rank 5 in a slot; its factors by (layer, name, piece), on the GPU in 64 bits."""
    g = torch.Generator(device=model.device).manual_seed(seed)
    found = {}
    for i, L in enumerate(model.layers):
        for name, a in L.adapters.items():
            factors = []
            for j, n in enumerate(a.pieces):
                if name not in names or (name == "w_qkv" and j == 1):  # (no adapter on k)
                    factors.append(None)
                    continue
                f = [(torch.randn(*s, device=model.device, generator=g) * std).to(torch.bfloat16)
                     for s, std in (((5, a.k), a.k ** -0.5), ((n, 5), 0.1 * size))]
                factors.append(f)
                found[i, name, j] = [t.double() for t in f]
            a.set(slot, factors, 1.5)
    return found


def _restated(model, ids, found=None):
    """The last position's logits, 64-bit arithmetic rounded where the engine rounds."""
    from minimal_inference_amd.mxfp8 import MXFP8

    cfg, found = model.cfg, found or {}
    bf = lambda t: t.to(torch.bfloat16).double()  # noqa: E731
    nq, nkv, d, t = cfg.num_attention_heads, cfg.num_key_value_heads, cfg.head_dim, len(ids)

    def rows8(h, w):
        if not isinstance(w, MXFP8):
            return bf(h)
        codes, scales = om8.quantize(h)
        return om8.values(codes, scales).to(h.device)

    def project(h, li, name, bias=None):
        w = getattr(model.layers[li], name)
        v = om8.values(w.codes, w.scales) if isinstance(w, MXFP8) else w.double()
        y = h @ v.t() + (0.0 if bias is None else bias.double())
        pieces = model.layers[li].adapters[name].pieces if found else []
        if any((li, name, j) in found for j in range(len(pieces))):
            parts = list(bf(y).split(pieces, 1))
            for j in range(len(pieces)):
                if (li, name, j) in found:
                    a, b = found[li, name, j]
                    parts[j] = parts[j] + 1.5 * (h @ a.t()) @ b.t()
            y = torch.cat(parts, 1)
        return y

    def rms(x, w):
        return x / (x.square().mean(-1, keepdim=True) + cfg.rms_norm_eps).sqrt() * w.double()

    x = model.embed[torch.tensor(ids, device=model.device)].double()
    cos, sin = model.cos[:t].double()[:, None], model.sin[:t].double()[:, None]
    rope = lambda v: bf(bf(v * cos) + bf(torch.cat((-v[..., d // 2:], v[..., : d // 2]), -1) * sin))  # noqa: E731
    for li, L in enumerate(model.layers):
        qkv = bf(project(rows8(rms(x, L.in_norm), L.w_qkv), li, "w_qkv", L.b_qkv)).view(t, nq + 2 * nkv, d)
        q, k, v = rope(qkv[:, :nq]), rope(qkv[:, nq: nq + nkv]), qkv[:, nq + nkv:]
        k, v = k.repeat_interleave(nq // nkv, 1), v.repeat_interleave(nq // nkv, 1)
        s = torch.matmul(q.transpose(0, 1), k.permute(1, 2, 0).contiguous()) * d ** -0.5
        s = s.masked_fill(torch.ones(t, t, device=s.device).triu(1).bool(), float("-inf"))
        o = bf(torch.matmul(torch.softmax(s, -1), v.transpose(0, 1).contiguous()).transpose(0, 1).reshape(t, nq * d))
        x = bf(x + bf(project(rows8(o, L.w_o), li, "w_o")))
        gate, up = project(rows8(rms(x, L.post_norm), L.w_gate_up), li, "w_gate_up").chunk(2, -1)
        x = bf(x + bf(project(rows8(gate * torch.sigmoid(gate) * up, L.w_down), li, "w_down")))
    return bf(rms(x[-1:], model.norm)) @ model.lm_head.double().t()


def _prompts(lens, seed=1):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 4096, (n,), generator=g).tolist() for n in lens]


def _off(got, want):
    return float((got.double() - want).abs().max() / want.abs().max())


@pytest.mark.parametrize("bias", [True, False])
def test_model_with_8_bit_layers(dev, bias):
    """Prefill logits of prompts of one to many rows, and a decode step's; fewer bytes."""
    from minimal_inference_amd.engine import Request, Scheduler
    from minimal_inference_amd.mxfp8 import MXFP8

    model = _model(dev, bias=bias)
    full = model.weight_bytes()
    model.quantize_weights("mxfp8")
    model.quantize_weights("mxfp8")  # (a second call leaves it as it is)
    assert model.weight_bytes() < full and all(isinstance(getattr(L, n), MXFP8) for L in model.layers for n in NAMES)
    for lens in ([1], [5, 40, 77], [200, 3]):
        prompts = _prompts(lens)
        sch = Scheduler(model, max_batch_size=4, max_seq_len=256, use_graphs=False, keep_logits=True)
        for i, ids in enumerate(prompts):
            sch.submit(Request(str(i), ids, 3, 0.0))
        sch.step()
        for i, ids in enumerate(prompts):
            assert _off(sch.p_logits[i], _restated(model, ids)) < BOUND_8_BIT
            token = sch.active[i].generated_tokens[0]
            assert _off(sch.d_logits[i], _restated(model, ids + [token])) < BOUND_8_BIT


@pytest.mark.parametrize("weight_format", ["bfloat16", "mxfp8"])
def test_adapters_of_a_batch(dev, weight_format):
    """Requests with different adapters, one of them without and two sharing one, in one batch: each row's
    prefill and decode logits are those of its own adapter, and another adapter's are far off."""
    from minimal_inference_amd.engine import Request, Scheduler

    bound = BOUND_8_BIT if weight_format == "mxfp8" else E2E_LOGIT_REL_BOUND
    model = _model(dev)
    model.enable_adapters(3, 8)
    assert model.adapter_slots == 3
    if weight_format == "mxfp8":
        model.quantize_weights("mxfp8")
    found = [_fill(model, s, 10 + s, size=3.0) for s in range(3)]
    prompts, slots = _prompts([9, 33, 70, 21, 4]), [1, -1, 0, 2, 1]
    sch = Scheduler(model, max_batch_size=5, max_seq_len=256, use_graphs=False, keep_logits=True)
    for i, (ids, s) in enumerate(zip(prompts, slots)):
        sch.submit(Request(str(i), ids, 3, 0.0, adapter=s))
    sch.step()
    for i, (ids, s) in enumerate(zip(prompts, slots)):
        mine = found[s] if s >= 0 else None
        want = _restated(model, ids, mine)
        assert _off(sch.p_logits[i], want) < bound
        assert _off(_restated(model, ids, found[(s + 1) % 3]), want) > 4 * E2E_LOGIT_REL_BOUND
        token = sch.active[i].generated_tokens[0]
        assert _off(sch.d_logits[i], _restated(model, ids + [token], mine)) < bound


@pytest.mark.parametrize("weight_format", ["bfloat16", "mxfp8"])
def test_scheduler_with_adapters(dev, weight_format):
    """Graphs (of batches with adapters and without), windows and pipelining against eager steps: requests
    come and go, so that batches shrink, and windows with and without adapters follow each other."""
    from minimal_inference_amd.engine import Request, Scheduler

    runs = []
    for options in ({"use_graphs": False}, {}, {"decode_window": 3, "pipeline": True}):
        model = _model(dev)
        model.enable_adapters(2, 8, ("w_qkv", "w_down"))
        if weight_format == "mxfp8":
            model.quantize_weights("mxfp8")
        for s in range(2):
            _fill(model, s, 20 + s, size=3.0)
        sch = Scheduler(model, max_batch_size=4, max_seq_len=256, **options)
        reqs = [Request(str(i), ids, 3 + 2 * (i % 4), 0.0, adapter=(-1, 0, 1, -1)[i % 4]) for i, ids in
                enumerate(_prompts([5, 18, 31, 44, 57, 7, 9]))]
        for r in reqs:
            sch.submit(r)
        sch.run()
        runs.append([r.generated_tokens for r in reqs])
    assert [len(t) for t in runs[0]] == [3 + 2 * (i % 4) for i in range(7)]
    assert runs[0] == runs[1] == runs[2]
    with pytest.raises(ValueError, match="adapter 2"):
        sch.submit(Request("x", [1], 1, 0.0, adapter=2))
    with pytest.raises(ValueError, match="adapter -2"):
        sch.submit_request(Request("x", [1], 1, 0.0, adapter=-2))


def test_model_refuses(dev):
    model = _model(dev)
    with pytest.raises(ValueError, match="weight_format"):
        model.quantize_weights("fp8")
    with pytest.raises(ValueError, match="any of"):
        model.enable_adapters(2, 8, ("w_x",))
    for slots, rank in ((0, 8), (1024, 8), (2, 7), (2, 136)):
        with pytest.raises(ValueError):
            model.enable_adapters(slots, rank)
        assert model.adapter_slots == 0
    model.enable_adapters(2, 8)
    with pytest.raises(ValueError, match="already"):
        model.enable_adapters(2, 8)
    model.quantize_weights("mxfp8")
    before = [getattr(L, n) for L in model.layers for n in NAMES]
    with pytest.raises(ValueError, match="another"):
        model.quantize_weights("mxfp4")
    assert all(a is b for a, b in zip(before, [getattr(L, n) for L in model.layers for n in NAMES]))
    unfused = _model(dev)
    unfused.fused_dense = False
    for call in (lambda: unfused.quantize_weights("mxfp8"), lambda: unfused.enable_adapters(1, 8)):
        with pytest.raises(ValueError, match="fused_dense"):
            call()


def test_unfused_layers_refuse_adapters(dev):
    """A model whose fused layers are switched off after adapters were enabled: requests without one run, one
    with an adapter is refused by the step, not served without it."""
    from minimal_inference_amd.engine import Request, Scheduler

    model = _model(dev)
    model.enable_adapters(1, 8)
    model.fused_dense = False
    sch = Scheduler(model, max_batch_size=2, max_seq_len=64, use_graphs=False)
    sch.submit(Request("a", [1, 2, 3], 2, 0.0))
    sch.run()
    sch.submit(Request("b", [1, 2, 3], 2, 0.0, adapter=0))
    with pytest.raises(ValueError, match="fused_dense"):
        sch.run()


def _write(path, tensors, **config):
    from safetensors.torch import save_file

    path.mkdir()
    (path / "adapter_config.json").write_text(json.dumps({"peft_type": "LORA", "r": 4, "lora_alpha": 10} | config))
    save_file(tensors, str(path / "adapter_model.safetensors"))
    return str(path)


def test_load_adapter(dev, tmp_path):
    """Factors and scale land in their slot; modules that a file lacks are cleared; a file that does not fit
    changes nothing."""
    from minimal_inference_amd.weights import load_adapter

    model = _model(dev)
    g = torch.Generator().manual_seed(4)
    key = "base_model.model.model.layers.{}.{}.lora_{}.weight"
    good = {key.format(1, "self_attn.v_proj", "A"): torch.randn(4, 256, generator=g),
            key.format(1, "self_attn.v_proj", "B"): torch.randn(128, 4, generator=g),
            key.format(2, "mlp.down_proj", "A"): torch.randn(4, 672, generator=g),
            key.format(2, "mlp.down_proj", "B"): torch.randn(256, 4, generator=g)}
    path = _write(tmp_path / "good", good)
    with pytest.raises(ValueError, match="room for 0"):
        load_adapter(model, 0, path)
    model.enable_adapters(2, 8, ("w_qkv", "w_down"))
    _fill(model, 1, 1)
    load_adapter(model, 1, path)
    a = model.layers[1].adapters["w_qkv"]
    assert float(a.scale[1]) == 2.5
    assert torch.equal(a.a[1, 16:20].cpu(), good[key.format(1, "self_attn.v_proj", "A")].to(torch.bfloat16))
    assert torch.equal(a.b[1, 384 + 128:, :4].cpu(), good[key.format(1, "self_attn.v_proj", "B")].to(torch.bfloat16))
    assert not bool(a.a[1, :16].any()) and not bool(a.a[1, 20:].any()) and not bool(a.b[1, : 384 + 128].any())
    assert not bool(model.layers[0].adapters["w_qkv"].a[1].any()) and bool(model.layers[2].adapters["w_down"].a[1].any())
    load_adapter(model, 0, _write(tmp_path / "rs", good, use_rslora=True))
    assert float(a.scale[0]) == 5.0
    held = [t.clone() for L in model.layers for x in L.adapters.values() for t in (x.a, x.b, x.scale)]
    lone = {key.format(1, "self_attn.v_proj", "A"): torch.zeros(4, 256)}  # (an A without its B)
    wide = {key.format(1, "self_attn.v_proj", "A"): torch.zeros(9, 256), key.format(1, "self_attn.v_proj", "B"): torch.zeros(128, 9)}
    bad = [(good | {key.format(1, "self_attn.o_proj", "A"): torch.zeros(4, 384)}, {}), (lone, {}), (wide, {"r": 9}), (good, {"r": 5}), (good, {"r": 0}),
           (good | {key.format(3, "mlp.down_proj", "A"): torch.zeros(4, 672)}, {}), (good | {"x.weight": torch.zeros(1)}, {}),
           (good, {"use_dora": True}), (good, {"bias": "all"}), (good, {"peft_type": "IA3"})]
    for i, (tensors, config) in enumerate(bad):
        with pytest.raises(ValueError):
            load_adapter(model, 1, _write(tmp_path / f"bad{i}", tensors, **config))
    for slot in (-1, 2):
        with pytest.raises(ValueError, match="room for 2"):
            load_adapter(model, slot, path)
    assert all(torch.equal(x, y) for x, y in zip(held, [t for L in model.layers for x in L.adapters.values() for t in (x.a, x.b, x.scale)]))


def test_checkpoint_is_not_loaded_into_8_bit_weights(dev, tmp_path):
    from minimal_inference_amd.weights import load_weights

    model = _model(dev)
    model.quantize_weights("mxfp8")
    with pytest.raises(ValueError, match="8-bit"):
        load_weights(model, str(tmp_path))


def test_server_engine_with_8_bit_layers_and_adapters(dev, tmp_path):
    """weight_format: mxfp8 and adapters in the server's configuration: the loop's greedy tokens are those of a
    scheduler over a model made by hand."""
    import queue

    from minimal_inference_amd.engine import Request, Scheduler
    from minimal_inference_amd.model import PRESETS, Model
    from minimal_inference_amd.mxfp8 import MXFP8
    from minimal_inference_amd.server import init_engine
    from minimal_inference_amd.weights import load_adapter

    g = torch.Generator().manual_seed(6)
    key = "base_model.model.model.layers.{}.self_attn.q_proj.lora_{}.weight"
    factors = {}
    for i in range(24):
        factors[key.format(i, "A")] = torch.randn(4, 896, generator=g) * 896 ** -0.5
        factors[key.format(i, "B")] = torch.randn(896, 4, generator=g)
    path = _write(tmp_path / "one", factors)
    sizes = {"max_batch_size": 4, "max_seq_len": 256}
    sch, _, _, stops = init_engine({"model_preset": "qwen2.5-0.5b", "weight_format": "mxfp8", "seed": 5, "scheduler": sizes,
                                    "adapters": {"one": path}, "adapter_rank": 8})
    prompt = list(range(40, 100))
    try:
        assert all(isinstance(getattr(L, n), MXFP8) for L in sch.model.layers for n in NAMES) and sch.adapter_slots == 1
        served = []
        for slot in (-1, 0):
            got: queue.Queue = queue.Queue()
            sch.submit_request(Request("a", prompt, 12, 0.0, adapter=slot, sink=got.put))
            served.append([])
            while (token := got.get(timeout=60)) is not None:
                served[-1].append(token)
    finally:
        sch.stop()
    model = Model(PRESETS["qwen2.5-0.5b"], dev, seed=5, max_positions=256 + 16)
    model.quantize_weights("mxfp8")
    model.enable_adapters(1, 8)
    load_adapter(model, 0, path)
    want = []
    for slot in (-1, 0):
        own = Scheduler(model, eos_token_ids=stops or None, **sizes)
        req = Request("b", prompt, 12, 0.0, adapter=slot)
        own.submit(req)
        own.run()
        want.append(req.generated_tokens)
    assert served == want and served[0] != served[1]
