"""GPU: rows without an adapter get the same bits whatever rows stand beside them, through a gated projection and through
a model; rows with one get SiLU(gate) * up of sums that are held in fp32 from the projection on.

Bars of rows with an adapter are those of test_gpu_adapters with the fp32 sums y as they are: fp32 additions start from
y, so each may lose 2^-24 of |y| and of the products added.
"""

from __future__ import annotations

import pytest
import torch

from oracle import mxfp8 as om8
from tests.test_gpu_model_8bit import _fill, _model, _prompts

pytestmark = pytest.mark.gpu

FORMATS = ["bfloat16", "mxfp4", "mxfp8"]


def _case(dev, rows, k, half, rank, slots, seed=0):
    from minimal_inference_amd.adapters import AdapterPlan, Adapters

    g = torch.Generator(device=dev).manual_seed(seed + rows + k)
    randn = lambda *s: torch.randn(*s, device=dev, generator=g)  # noqa: E731
    ad = Adapters((randn(slots, 2 * rank, k) * k ** -0.5).to(torch.bfloat16), randn(slots, 2 * half, rank).to(torch.bfloat16),
                  0.25 + torch.rand(slots, device=dev, generator=g), [half, half])
    slot = (torch.arange(rows, device=dev) % (slots + 1) - 1).to(torch.int32)
    plan = AdapterPlan(rows, slots, dev)
    plan.plan(slot)
    x = randn(rows, k).to(torch.bfloat16)
    w = (randn(2 * half, k) * 2 * k ** -0.5).to(torch.bfloat16)
    return x, w, ad, slot, plan


def _sums(values, ad, slot, y, rows):
    """Gate and up of y and the rows' adapters in 64 bits, and how far the kernel's may be from them."""
    ref, tol = y.double()[rows], torch.zeros_like(y, dtype=torch.float64)[rows]
    k, rank, half = ad.k, ad.rank, ad.pieces[0]
    for i, row in enumerate(rows.tolist()):
        s = int(slot[row])
        a, b, scale = ad.a[s].double(), ad.b[s].double(), ad.scale[s].double()
        v = a @ values[row] * scale
        ev = 4 * k ** 0.5 * 2.0 ** -24 * (a.abs() @ values[row].abs()) * scale + (2.0 ** -16 + 2.0 ** -24) * v.abs()
        for j in range(2):
            part, cols = slice(j * rank, (j + 1) * rank), slice(j * half, (j + 1) * half)
            w = b[cols]
            size = ref[i, cols].abs() + w.abs() @ v[part].abs()
            ref[i, cols] += w @ v[part]
            tol[i, cols] = w.abs() @ ev[part] + (2 * rank + 2) * 2.0 ** -24 * size
    return ref[:, :half], ref[:, half:], tol[:, :half], tol[:, half:]


def _want(*args):
    """SiLU(gate) * up of those, and how far a value may be from it before its rounding."""
    G, U, dg, du = _sums(*args)
    want = G * torch.sigmoid(G) * U
    return want, 1.1 * dg * (U.abs() + du) + G.abs() * du + 2.0 ** -20 * want.abs()


# few rows, blocks that share k, blocks, the largest blocks, rows behind the last whole block; ranks of every size of launch
SIZES = [(1, 256, 96, 8, 1), (5, 896, 4864, 16, 3), (33, 4096, 672, 24, 4), (64, 1056, 96, 64, 5), (130, 8192, 128, 16, 3), (200, 512, 352, 32, 7),
         (300, 896, 992, 128, 2), (333, 256, 4864, 16, 9), (1030, 1024, 2048, 64, 3)]


def _sample(slot):
    """Some rows with an adapter."""
    rows = (slot >= 0).nonzero()[:, 0]
    return rows[:: max(1, len(rows) // 12)]


@pytest.mark.parametrize("rows,k,half,rank,slots", SIZES)
def test_8_bit(dev, rows, k, half, rank, slots):
    from minimal_inference_amd.adapters import add_adapters_silu
    from minimal_inference_amd.mxfp8 import gate_up_mxfp8, linear_silu_mxfp8, quantize_mxfp8

    x, w, ad, slot, plan = _case(dev, rows, k, half, rank, slots)
    m, w8 = quantize_mxfp8(x), quantize_mxfp8(w)
    room = torch.full((rows, 2 * half + 8), 7.0, device=dev)
    y = gate_up_mxfp8(m, w8, out=room[:, 4: 4 + 2 * half])
    assert bool((room[:, :4] == 7).all()) and bool((room[:, 4 + 2 * half:] == 7).all())
    base = linear_silu_mxfp8(m, w8, quantize=True)
    before = y.clone()
    q = add_adapters_silu(y, m, ad, plan, quantize=True)
    assert torch.equal(y, before)
    none = slot < 0
    assert torch.equal(q.codes.view(torch.uint8)[none], base.codes.view(torch.uint8)[none])
    assert torch.equal(q.scales[none], base.scales[none])
    # (one sum of 8-bit products is within 2^-10 of the 2-norm of its products, as in test_gpu_mxfp8)
    vx, vw = om8.values(m.codes, m.scales).to(dev), om8.values(w8.codes, w8.scales).to(dev)
    assert bool(((y.double() - vx @ vw.t()).abs() <= 2.0 ** -10 * (vx.square() @ vw.square().t()).sqrt()).all())
    some = _sample(slot)
    want, near = _want(vx, ad, slot, y, some)
    unit = torch.exp2(q.scales.double() - 127.0).repeat_interleave(32, 1)[some]
    got = om8.values(q.codes, q.scales).to(dev)[some]
    assert bool(((got - want).abs() <= near + ((want.abs() + near) * 2.0 ** -4).maximum(unit * 2.0 ** -10)).all())


@pytest.mark.parametrize("rows,k,half,rank,slots", SIZES)
def test_4_bit(dev, rows, k, half, rank, slots):
    from minimal_inference_amd.adapters import add_adapters_silu
    from minimal_inference_amd.mxfp4 import gate_up_mxfp4, linear_silu_mxfp4, quantize_mxfp4

    x, w, ad, slot, plan = _case(dev, rows, k, half, rank, slots)
    w4 = quantize_mxfp4(w)
    none, some = slot < 0, _sample(slot)
    room = torch.full((rows, 2 * half + 8), 7.0, device=dev)
    y = gate_up_mxfp4(x, w4, out=room[:, 4: 4 + 2 * half])
    assert bool((room[:, :4] == 7).all()) and bool((room[:, 4 + 2 * half:] == 7).all())
    out = add_adapters_silu(y, x, ad, plan)
    assert torch.equal(out[none], linear_silu_mxfp4(x, w4)[none])
    want, near = _want(x.double(), ad, slot, y, some)
    assert bool(((out[some].double() - want).abs() <= near + 2 ** -8 * (want.abs() + near)).all())
    # 4-bit rows beside 4-bit weights (the adapters read the bf16 rows)
    x4 = quantize_mxfp4(x)
    out = add_adapters_silu(gate_up_mxfp4(x4, w4), x, ad, plan)
    assert torch.equal(out[none], linear_silu_mxfp4(x4, w4)[none])


@pytest.mark.parametrize("rows,k,half,rank,slots", SIZES)
def test_bf16(dev, rows, k, half, rank, slots):
    """Every step rounded to bf16, 2^-8 each: the sums, silu (whose slope is 1.1 at most) and the product.  (The same
    steps by add_adapters and silu_mul may differ in bits: add_adapters of few rows sums in another order.)"""
    from minimal_inference_amd.adapters import add_adapters_silu
    from minimal_inference_amd.dense import linear, linear_silu

    x, w, ad, slot, plan = _case(dev, rows, k, half, rank, slots)
    y = linear(x, w)
    out = add_adapters_silu(y, x, ad, plan, stepwise=True)
    assert torch.equal(out[slot < 0], linear_silu(x, w)[slot < 0])
    some = _sample(slot)
    G, U, dg, du = _sums(x.double(), ad, slot, y, some)
    dg, du = dg + 2 ** -8 * (G.abs() + dg), du + 2 ** -8 * (U.abs() + du)
    silu = G * torch.sigmoid(G)
    ds = 1.1 * dg + 2.0 ** -22 * silu.abs()
    ds = ds + 2 ** -8 * (silu.abs() + ds)
    want, near = silu * U, ds * (U.abs() + du) + silu.abs() * du
    assert bool(((out[some].double() - want).abs() <= near + 2 ** -8 * (want.abs() + near)).all())


@pytest.mark.parametrize("layer", FORMATS)
def test_gated_projection_replayed(dev, layer):
    """A captured projection and its adapters under several plans of as many rows, and NaN under one of another
    number."""
    from minimal_inference_amd.adapters import add_adapters_silu
    from minimal_inference_amd.dense import linear
    from minimal_inference_amd.mxfp4 import gate_up_mxfp4, quantize_mxfp4
    from minimal_inference_amd.mxfp8 import gate_up_mxfp8, quantize_mxfp8

    x, w, ad, slot, plan = _case(dev, 130, 8192, 128, 16, 3)
    if layer == "mxfp8":
        rows, weight = quantize_mxfp8(x), quantize_mxfp8(w)
        call = lambda: add_adapters_silu(gate_up_mxfp8(rows, weight), rows, ad, plan, quantize=True).dequantize()  # noqa: E731
    elif layer == "mxfp4":
        weight = quantize_mxfp4(w)
        call = lambda: add_adapters_silu(gate_up_mxfp4(x, weight), x, ad, plan)  # noqa: E731
    else:
        call = lambda: add_adapters_silu(linear(x, w), x, ad, plan, stepwise=True)  # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for i in range(4):
        plan.plan(slot.roll(i))
        graph.replay()
        assert torch.equal(got, call())
        plan.plan(slot[:99])
        graph.replay()
        assert bool(got.isnan().all())


def _run(model, prompts, slots, **options):
    from minimal_inference_amd.engine import Request, Scheduler

    sch = Scheduler(model, max_batch_size=len(prompts), max_seq_len=256, keep_logits=True, **options)
    reqs = [Request(str(i), ids, 4, 0.0, adapter=s) for i, (ids, s) in enumerate(zip(prompts, slots))]
    for r in reqs:
        sch.submit(r)
    sch.step()
    logits = [sch.p_logits.clone()]
    while sch.has_work():
        logits.append(sch.d_logits.clone())
        sch.step()
    return logits, [r.generated_tokens for r in reqs]


@pytest.mark.parametrize("use_graphs", [False, True])
@pytest.mark.parametrize("layer", FORMATS)
@pytest.mark.parametrize("lens", [[9, 33, 70, 21, 4], [200, 3, 150]])  # (prefills of 137 and 353 rows)
def test_a_request_without_an_adapter_beside_others(dev, layer, lens, use_graphs):
    """All four projections have adapters: the requests without one have the logits of a batch without any, bit for
    bit, in prefill and decode; the others' are other logits."""
    model = _model(dev)
    model.enable_adapters(3, 8)
    if layer != "bfloat16":
        model.quantize_weights(layer)
    for s in range(3):
        _fill(model, s, 10 + s, size=3.0)
    prompts = _prompts(lens)
    slots = [(-1, 0, 2, -1, 1)[i] for i in range(len(lens))]
    alone, tokens = _run(model, prompts, [-1] * len(lens), use_graphs=use_graphs)
    mixed, beside = _run(model, prompts, slots, use_graphs=use_graphs)
    for a, b in zip(alone, mixed):
        for i, s in enumerate(slots):
            assert torch.equal(a[i], b[i]) == (s < 0), i
    assert all(t == u for t, u, s in zip(tokens, beside, slots) if s < 0)


@pytest.mark.parametrize("layer", FORMATS)
def test_scheduler_with_adapters_beside_every_projection(dev, layer):
    """Graphs, windows and pipelining against eager steps, as requests come and go."""
    from minimal_inference_amd.engine import Request, Scheduler

    runs = []
    for options in ({"use_graphs": False}, {}, {"decode_window": 3, "pipeline": True}):
        model = _model(dev)
        model.enable_adapters(2, 8)
        if layer != "bfloat16":
            model.quantize_weights(layer)
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
