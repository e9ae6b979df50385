"""GPU: the operators around attention used together, as a decode step and a server do.

A block with norms on either side and 4-bit projections, down to the drawn id, eager and
captured; the model with 4-bit layers against the same model on the values that these
layers stand for; a scheduler over it.
"""

from __future__ import annotations

import pytest
import torch

from oracle.draw import draw_row

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 5, 48, 100])
@pytest.mark.parametrize("acts", ["bf16", "mxfp4"])
def test_block_to_token(dev, rows, acts):
    """x -> norm -> gate, up and down in 4 bits -> norm, gate, scale, sum, norm -> LM
    head -> draw.  Each operator against its own 64-bit form on the inputs it got is its
    own tests' matter; here the chain, replayed on new inputs, gives the eager bits, and
    ids are the oracle's draws from the chain's logits."""
    from minimal_inference_amd.dense import add_rms_norm, linear, post_norm_add_rms_norm
    from minimal_inference_amd.mxfp4 import linear_mxfp4, linear_silu_mxfp4, quantize_mxfp4
    from minimal_inference_amd.sampling import Sampler

    hidden, inter, vocab = 512, 1184, 5000
    g = torch.Generator(device=dev).manual_seed(rows)

    def randn(*shape, std=1.0):
        return (std * torch.randn(*shape, device=dev, generator=g)).to(torch.bfloat16)

    gate_up, down = quantize_mxfp4(randn(2 * inter, hidden, std=0.05)), quantize_mxfp4(randn(hidden, inter, std=0.05))
    head, norms = randn(vocab, hidden, std=0.1), [1 + randn(hidden, std=0.1) for _ in range(3)]
    gate = randn(hidden)
    x, u = randn(rows, hidden), torch.rand(rows, device=dev, generator=g)
    s = Sampler(dev, rows, vocab=vocab)
    s.set_params([0.8] * rows, [0.95] * rows, top_k=[100] * rows, min_p=[0.01] * rows)
    make = quantize_mxfp4 if acts == "mxfp4" else (lambda t: t)

    def step():
        stream = torch.empty_like(x)
        h = add_rms_norm(x, None, norms[0], 1e-6, write_x=False)
        y = linear_mxfp4(make(linear_silu_mxfp4(make(h), gate_up)), down)
        h = post_norm_add_rms_norm(x, y, norms[1], norms[2], 1e-6, gate=gate, scale=0.5, x_out=stream)
        logits = linear(h, head)
        return stream, h, logits, s.draw(logits, u, out=torch.empty(rows, dtype=torch.int64, device=dev))

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    f = lambda v: torch.tensor(v).double().item()  # noqa: E731
    for seed in range(3):
        x.copy_(torch.randn(rows, hidden, generator=torch.Generator().manual_seed(seed)))
        u.copy_(torch.rand(rows, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        held = [t.clone() for t in got]
        assert all(torch.equal(a, b) for a, b in zip(held, step()))
        logits = held[2].cpu()
        assert held[3].tolist() == [draw_row(logits[i], u[i].item(), f(0.8), 100, f(0.95), f(0.01)) for i in range(rows)]
        # the chain in 64 bits: each of its bf16 roundings is 2^-8 at most, and four of
        # them (h, the gated product, y and the stream) reach x_out; rows in 4 bits are
        # another function of h, so they are compared as bits alone
        if acts == "bf16":
            xd = x.double()
            rms = lambda t, w: t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-6) * w.double()  # noqa: E731
            a, b = (rms(xd, norms[0]) @ gate_up.dequantize().double().t()).chunk(2, -1)
            y = (a * torch.sigmoid(a) * b) @ down.dequantize().double().t()
            want = xd + 0.5 * gate.double() * rms(y, norms[1])
            assert float((held[0].double() - want).norm() / want.norm()) < 4 * 2 ** -8


def _small(dev, seed=3):
    from minimal_inference_amd.model import Model, ModelConfig

    cfg = ModelConfig(hidden_size=256, num_attention_heads=7, num_key_value_heads=1, head_dim=64, num_hidden_layers=3,
                      intermediate_size=672, vocab_size=4096, max_position_embeddings=512)
    return Model(cfg, dev, seed=seed, max_positions=512)


def test_model_with_4_bit_layers(dev):
    """Prefill and decode logits of the model with 4-bit layers are those of the bf16
    model on the values that the layers stand for, within the roundings of a few layers
    (both sides round the same products to bf16; their sums differ in order): relative
    2e-2 as between the fused and unfused kernels.  It holds fewer bytes."""
    from minimal_inference_amd.engine import Request, Scheduler

    logits, tokens, sizes = [], [], []
    for four in (True, False):
        model = _small(dev)
        full = model.weight_bytes()
        model.quantize_weights()
        sizes.append((full, model.weight_bytes()))
        if not four:
            for L in model.layers:
                for name in ("w_qkv", "w_o", "w_gate_up", "w_down"):
                    setattr(L, name, getattr(L, name).dequantize())
        sch = Scheduler(model, max_batch_size=4, max_seq_len=256, use_graphs=False, keep_logits=True)
        g = torch.Generator().manual_seed(1)
        for i, n in enumerate([5, 40, 77]):
            sch.submit(Request(str(i), torch.randint(0, 4096, (n,), generator=g).tolist(), 3, 0.0))
        sch.step()
        logits.append([sch.p_logits[:3].float().clone(), sch.d_logits[:3].float().clone()])
        tokens.append([r.generated_tokens[0] for r in sch.active])
    # (a prompt whose two best ids are closer than that may go on with either)
    alike = [i for i, (a, b) in enumerate(zip(*tokens)) if a == b]
    assert alike
    for (a, b), rows in zip(zip(*logits), (range(3), alike)):
        for i in rows:
            assert float((a[i] - b[i]).abs().max() / b[i].abs().max()) < 2e-2
    assert sizes[0][1] < sizes[0][0]


def test_scheduler_over_4_bit_layers(dev):
    """Graphs, whose batches are padded, and eager steps give the same tokens: up to 16
    rows, a row's result does not depend on the others."""
    from minimal_inference_amd.engine import Request, Scheduler

    runs = []
    for graphs in (True, False):
        model = _small(dev)
        model.quantize_weights()
        model.quantize_weights()  # (a second call leaves it as it is)
        sch = Scheduler(model, max_batch_size=8, max_seq_len=256, use_graphs=graphs)
        g = torch.Generator().manual_seed(2)
        reqs = [Request(str(i), torch.randint(0, 4096, (5 + 13 * i,), generator=g).tolist(), 4 + i, 0.0) for i in range(7)]
        for r in reqs:
            sch.submit(r)
        sch.run()
        runs.append([r.generated_tokens for r in reqs])
    assert [len(t) for t in runs[0]] == [4 + i for i in range(7)]
    assert runs[0] == runs[1]


def test_refuses_unfused(dev):
    from minimal_inference_amd.model import Model

    model = _small(dev)
    model.fused_dense = False
    with pytest.raises(ValueError):
        model.quantize_weights()


def test_matrices_past_32_bits(dev):
    """More than 2^32 bytes of rows, of codes and of output: the last rows are those of
    the same rows alone."""
    from minimal_inference_amd.dense import post_norm_add_rms_norm
    from minimal_inference_amd.mxfp4 import MXFP4, linear_mxfp4, quantize_mxfp4

    rows, cols = 600_000, 4096
    g = torch.Generator(device=dev).manual_seed(0)
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device=dev).normal_(generator=g)
    q = quantize_mxfp4(x)
    back = q.dequantize()
    for part in (slice(0, 40), slice(rows - 40, rows)):
        assert torch.equal(back[part], quantize_mxfp4(x[part]).dequantize())
    del q
    w = torch.ones(cols, dtype=torch.bfloat16, device=dev)
    tail = slice(rows - 40, rows)
    want_x = torch.empty(40, cols, dtype=torch.bfloat16, device=dev)
    want_h = post_norm_add_rms_norm(x[tail], back[tail], w, w, 1e-6, x_out=want_x)
    h = post_norm_add_rms_norm(x, back, w, w, 1e-6, h_out=back)
    assert torch.equal(x[tail], want_x) and torch.equal(h[tail], want_h)
    del x, back, h
    # whole numbers: the sums are exact, whatever the form of the launch
    values = torch.tensor([0, 1, 2, 3, 4, 6, -1, -2, -3, -4, -6], dtype=torch.bfloat16, device=dev)
    for rows, n, k in ((270_000, 10_240, 64), (3, 1 << 20, 8192)):
        x = values[torch.randint(0, 11, (rows, k), device=dev, generator=g)]
        x[:, ::32] = 6.0
        wc = torch.randint(0, 256, (n, k // 2), device=dev, generator=g, dtype=torch.uint8)
        weight = MXFP4.from_codes(wc, torch.full((n, k // 32), 128, dtype=torch.uint8, device=dev))
        one = MXFP4.from_codes(wc[-50:].contiguous(), torch.full((50, k // 32), 128, dtype=torch.uint8, device=dev))
        ref = (x[-40:].double() @ one.dequantize().double().t()).to(torch.bfloat16)
        for a in (x, quantize_mxfp4(x)):
            assert torch.equal(linear_mxfp4(a, weight)[-40:, -50:], ref)


def test_draws_from_rows_far_apart(dev):
    from minimal_inference_amd.sampling import Sampler

    b, v, apart = 40, 32768, 1 << 26
    wide = torch.empty(b * apart, dtype=torch.bfloat16, device=dev)
    logits = wide.as_strided((b, v), (apart, 1))
    logits.normal_(std=3.0, generator=torch.Generator(device=dev).manual_seed(1))
    u = torch.rand(b, device=dev, generator=torch.Generator(device=dev).manual_seed(2))
    s = Sampler(dev, b, vocab=v)
    s.set_params([0.8] * b, [0.95] * b, top_k=[100] * b, min_p=[0.01] * b)
    near = s.draw(logits.contiguous(), u).clone()
    assert torch.equal(s.draw(logits, u), near)


def test_server_engine_with_4_bit_layers(dev):
    """weight_format: mxfp4 in the server's configuration: the loop's greedy tokens are
    those of a scheduler over the same model quantised by hand."""
    import queue

    from minimal_inference_amd.engine import Request, Scheduler
    from minimal_inference_amd.model import PRESETS, Model
    from minimal_inference_amd.mxfp4 import MXFP4
    from minimal_inference_amd.server import init_engine

    sizes = {"max_batch_size": 4, "max_seq_len": 256}
    sch, _, _, stops = init_engine({"model_preset": "qwen2.5-0.5b", "weight_format": "mxfp4", "seed": 5, "scheduler": sizes})
    try:
        assert all(isinstance(w, MXFP4) for layer in sch.model.layers
                   for w in (layer.w_qkv, layer.w_o, layer.w_gate_up, layer.w_down))
        prompt = list(range(40, 100))
        got: queue.Queue = queue.Queue()
        sch.submit_request(Request("a", prompt, 12, 0.0, sink=got.put))
        served = []
        while (token := got.get(timeout=60)) is not None:
            served.append(token)
    finally:
        sch.stop()
    model = Model(PRESETS["qwen2.5-0.5b"], dev, seed=5, max_positions=256 + 16)
    model.quantize_weights()
    other = Scheduler(model, eos_token_ids=stops or None, seed=5, **sizes)
    request = Request("b", prompt, 12, 0.0)
    other.submit(request)
    other.run()
    assert served == request.generated_tokens
