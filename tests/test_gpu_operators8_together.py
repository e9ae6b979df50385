"""GPU: the 8-bit and adapter operators in a run of their own, as a layer uses them: eager, on a stream of
its own, two runs at once, captured and replayed; each form of the products; matrices past 32 bits.

Bars against 64 bits: products of whole numbers are exact in fp32, so their outputs are the nearest bf16 of
the exact value.  Replays and other streams repeat the eager run's bits: no sum's order depends on time.
"""

from __future__ import annotations

import pytest
import torch

from oracle import mxfp8 as om8

pytestmark = pytest.mark.gpu


class _Layer:
    """Two norms, the projections of an MLP and of q, k and v, adapters beside them."""

    def __init__(self, dev, hidden=448, inter=1120, slots=3, rank=8, seed=0):
        from minimal_inference_amd.adapters import Adapters
        from minimal_inference_amd.mxfp8 import quantize_mxfp8

        g = torch.Generator(device=dev).manual_seed(seed)
        rand = lambda *s, std=1.0: (torch.randn(*s, device=dev, generator=g) * std).to(torch.bfloat16)  # noqa: E731
        self.norm = rand(hidden)
        self.qkv = quantize_mxfp8(rand(hidden + 128, hidden, std=hidden ** -0.5))
        self.gate_up = quantize_mxfp8(rand(2 * inter, hidden, std=hidden ** -0.5))
        self.down = quantize_mxfp8(rand(hidden, inter, std=inter ** -0.5))
        make = lambda k, pieces: Adapters(rand(slots, len(pieces) * rank, k, std=k ** -0.5), rand(slots, sum(pieces), rank),  # noqa: E731
                                          torch.rand(slots, device=dev, generator=g), pieces)
        self.on_qkv, self.on_down = make(hidden, [hidden, 64, 64]), make(inter, [hidden])
        self.slots = slots

    def run(self, x, delta, plan):
        """(x + delta, q k v with adapters, the MLP's output with adapters); x is written."""
        from minimal_inference_amd.adapters import add_adapters
        from minimal_inference_amd.mxfp8 import add_rms_norm_mxfp8, linear_mxfp8, linear_silu_mxfp8

        h = add_rms_norm_mxfp8(x, delta, self.norm, 1e-6)
        qkv = add_adapters(linear_mxfp8(h, self.qkv), h, self.on_qkv, plan)
        act = linear_silu_mxfp8(h, self.gate_up, quantize=True)
        return x, qkv, add_adapters(linear_mxfp8(act, self.down), act, self.on_down, plan)


def _inputs(dev, rows, slots, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    x, d = (torch.randn(rows, 448, device=dev, generator=g).to(torch.bfloat16) for _ in range(2))
    return x, d, torch.randint(-1, slots, (rows,), device=dev, generator=g, dtype=torch.int32)


def _plan(dev, slot, slots, rows=None):
    from minimal_inference_amd.adapters import AdapterPlan

    plan = AdapterPlan(rows or slot.shape[0], slots, dev)
    plan.plan(slot)
    return plan


@pytest.mark.parametrize("rows", [1, 17, 300])
def test_a_layer_in_64_bits(dev, rows):
    """Outputs against the same quantities in 64 bits from the kernels' own codes on: each bar is a half step of
    bf16 per rounding plus the matrix instruction's cut (1.5e-5 of the largest sums' terms) and fp32 sums."""
    layer = _Layer(dev)
    x, d, slot = _inputs(dev, rows, 3, rows)
    plan = _plan(dev, slot, 3)
    from minimal_inference_amd.mxfp8 import add_rms_norm_mxfp8, linear_silu_mxfp8

    x0 = x.clone()
    got_x, qkv, y = layer.run(x, d, plan)
    total = (x0.double() + d.double())
    assert got_x is x and torch.equal(x, total.to(torch.bfloat16))
    h = add_rms_norm_mxfp8(x0, d, layer.norm, 1e-6)
    act = linear_silu_mxfp8(h, layer.gate_up, quantize=True)
    for got, rows8, w, a in ((qkv, h, layer.qkv, layer.on_qkv), (y, act, layer.down, layer.on_down)):
        v, wv = (om8.values(m.codes, m.scales).to(dev) for m in (rows8, w))
        base = v @ wv.t()
        size = v.abs() @ wv.abs().t()
        low = [torch.zeros_like(base) for _ in range(2)]
        for s in range(3):
            mine = (slot == s).nonzero()[:, 0]
            column = 0
            for i, n in enumerate(a.pieces):
                A = a.a[s, i * a.rank: (i + 1) * a.rank].double()
                B = a.b[s, column: column + n].double()
                scale = float(a.scale[s])
                low[0][mine, column: column + n] = scale * (v[mine] @ A.t()) @ B.t()
                low[1][mine, column: column + n] = scale * (v[mine].abs() @ A.abs().t()) @ B.abs().t()
                column += n
        want = base + low[0]
        # y to bf16 before the adapters add (2^-8), the sum to bf16 (2^-8), the middle values to bf16 (2^-8 of
        # their product's absolute sum), the cut, and fp32 sums of up to 1,120 terms (2^-24 each)
        bar = 2.0 ** -8 * (base.abs() + want.abs() + low[1]) * (1 + 2.0 ** -7) + (1.5e-5 + 1120 * 2.0 ** -24) * (size + low[1])
        assert bool(((got.double() - want).abs() <= bar).all())


@pytest.mark.parametrize("rows", [3, 130])
def test_replays_and_streams(dev, rows):
    """A graph replayed with new inputs and new slots, with eager runs between; a run on a stream of its own;
    two runs at once on two streams: all the bits of eager runs one by one."""
    layer = _Layer(dev)
    cases = [_inputs(dev, rows, 3, s) for s in range(4)]
    want = [[t.clone() for t in layer.run(x.clone(), d, _plan(dev, s, 3))] for x, d, s in cases]
    x, d, slot = (t.clone() for t in cases[0])
    plan = _plan(dev, slot, 3, rows + 5)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        got = layer.run(cases[1][0].clone(), cases[1][1], _plan(dev, cases[1][2], 3))
        layer.run(x.clone(), d, plan)
    torch.cuda.current_stream(dev).wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want[1]))
    graphs = []
    for _ in range(2):  # (two graphs over the same inputs)
        graph = torch.cuda.CUDAGraph()
        held = x.clone()
        with torch.cuda.graph(graph):
            plan.plan(slot)
            held.copy_(x)
            out = layer.run(held, d, plan)
        graphs.append((graph, out))
    for turn in range(6):
        i = turn % 4
        for t, new in zip((x, d, slot), cases[i]):
            t.copy_(new)
        graph, out = graphs[turn % 2]
        graph.replay()
        between = layer.run(cases[(i + 1) % 4][0].clone(), cases[(i + 1) % 4][1], _plan(dev, cases[(i + 1) % 4][2], 3))
        torch.cuda.synchronize(dev)
        assert all(torch.equal(a, b) for a, b in zip(out, want[i]))
        assert all(torch.equal(a, b) for a, b in zip(between, want[(i + 1) % 4]))
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    inputs = [(cases[i][0].clone(), cases[i][1], _plan(dev, cases[i][2], 3)) for i in (2, 3)]
    torch.cuda.synchronize(dev)
    outs = [[], []]
    for _ in range(8):
        for j in range(2):
            with torch.cuda.stream(streams[j]):
                a, b, p = inputs[j]
                held = a.clone()
                outs[j].append(layer.run(held, b, p))
    torch.cuda.synchronize(dev)
    assert all(torch.equal(a, b) for j in range(2) for o in outs[j] for a, b in zip(o, want[j + 2]))


@pytest.mark.parametrize("rows,other", [(3, 2), (3, 5), (600, 40), (40, 600)])
def test_replay_after_another_batch(dev, rows, other):
    """A replay after a plan of another number of rows gives NaN, everywhere and nowhere else, and after
    its own the eager bits again."""
    from minimal_inference_amd.adapters import AdapterPlan, add_adapters

    layer = _Layer(dev)
    x, y, slot = _inputs(dev, max(rows, other), 3, 1)
    y = y.repeat(1, 2)[:, : 448 + 128].contiguous()
    plan = AdapterPlan(max(rows, other), 3, dev)
    room = torch.full((rows + 2, 448 + 128 + 8), 7.0, dtype=torch.bfloat16, device=dev)
    out = room[1: rows + 1, : 448 + 128]
    run = lambda: add_adapters(y[:rows], x[:rows], layer.on_qkv, plan, out=out)  # noqa: E731
    plan.plan(slot[:rows])
    want = run().clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for _ in range(3):
        plan.plan(slot[:other])
        graph.replay()
        assert bool(out.isnan().all())
        with pytest.raises(ValueError, match="the plan is of"):
            run()
        plan.plan(slot[:rows])
        graph.replay()
        assert torch.equal(out, want)
    assert bool((room[0] == 7).all() and (room[-1] == 7).all() and (room[:, 448 + 128:] == 7).all())


def test_norms_past_fp32(dev):
    """Norms that fp32 does not hold make their block NaN, and leave the others as they are."""
    from minimal_inference_amd.mxfp8 import add_rms_norm_mxfp8

    g = torch.Generator(device=dev).manual_seed(3)
    x = torch.randn(4, 256, device=dev, generator=g).to(torch.bfloat16)
    w = torch.randn(256, device=dev, generator=g).to(torch.bfloat16)
    x[:, 40] = torch.tensor([4.0, -4.0, 8.0, -8.0], dtype=torch.bfloat16, device=dev)  # (times w: an infinity of either sign)
    want = add_rms_norm_mxfp8(x, None, w, 1e-6)
    w2 = w.clone()
    w2[40] = 3e38
    got = add_rms_norm_mxfp8(x, None, w2, 1e-6)
    assert bool((got.scales[:, 1] == 255).all()) and not bool(got.codes[:, 32:64].view(torch.uint8).any())
    for a, b in ((got.scales, want.scales), (got.codes.view(torch.uint8), want.codes.view(torch.uint8))):
        width = a.shape[1] // 8
        assert torch.equal(a[:, :width], b[:, :width]) and torch.equal(a[:, 2 * width:], b[:, 2 * width:])


def _whole(dev, rows, k, seed):
    """Whole numbers of -3..3 as MXFP8 with scales 1, 2 and 4, but the exact values' sums below 2^24."""
    from minimal_inference_amd.mxfp8 import MXFP8

    g = torch.Generator(device=dev).manual_seed(seed)
    m = MXFP8(rows, k, dev)
    m.codes.copy_(torch.randint(-3, 4, (rows, k), device=dev, generator=g).float().to(torch.float8_e4m3fn))
    m.scales.copy_(torch.randint(127, 130, (rows, k // 32), device=dev, generator=g, dtype=torch.uint8))
    return m


def _values32(m):
    """The same values in fp32, which holds them and their products' sums exactly (k * 12 * 12 < 2^24)."""
    return m.codes.float() * torch.exp2(m.scales.float() - 127.0).repeat_interleave(32, 1)


# rows, n, k: by the kernel's forms. Few rows: 1..64 by counts of 16 and of waves over k, alone and sharing k; blocks of 128 x 128, whole and
# split over k; blocks of 256 x 256, alone, with rows behind them as few rows, as a block, and with ragged columns and k.
FORMS = [(1, 33, 32), (1, 4864, 896), (7, 100, 14336), (16, 28672, 512), (17, 20000, 96), (31, 1000, 4128), (48, 257, 8192), (64, 30000, 128),
         (40, 40000, 96), (33, 82000, 64), (33, 4099, 12320), (20, 8192, 16416), (64, 3584, 18944), (47, 100, 8192),
         (65, 48, 32), (65, 129, 8224), (200, 1000, 544), (300, 2048, 18944), (1024, 4096, 512),
         (2048, 1056, 8192), (2057, 8192, 1024), (4096, 4112, 288), (4200, 4096, 1056), (2304, 8193, 4096), (8201, 2048, 4064)]


@pytest.mark.parametrize("rows,n,k", FORMS)
def test_forms_exactly(dev, rows, n, k):
    """Whole numbers: the products are exact, plain and with a bias; the rows and columns around out stay."""
    from minimal_inference_amd.mxfp8 import linear_mxfp8

    x, w = _whole(dev, rows, k, rows), _whole(dev, n, k, n)
    g = torch.Generator(device=dev).manual_seed(k)
    bias = torch.randint(-64, 65, (n,), device=dev, generator=g).to(torch.bfloat16)
    want = _values32(x) @ _values32(w).t()
    room = torch.full((rows + 2, n + 7), 7.0, dtype=torch.bfloat16, device=dev)
    linear_mxfp8(x, w, bias, out=room[1: rows + 1, :n])
    assert torch.equal(room[1: rows + 1, :n], (want + bias.float()).to(torch.bfloat16))
    assert bool((room[0] == 7).all() and (room[-1] == 7).all() and (room[:, n:] == 7).all())
    assert torch.equal(linear_mxfp8(x, w), want.to(torch.bfloat16))


@pytest.mark.parametrize("rows,n,k", [(64, 3584, 18944), (33, 4099, 12320), (300, 200, 4128)])
def test_without_a_workspace(dev, monkeypatch, rows, n, k):
    """Without room for parts the same sums, by workgroups that share nothing."""
    from minimal_inference_amd import mxfp8

    x, w = _whole(dev, rows, k, 1), _whole(dev, n, k, 2)
    assert mxfp8._workspace_size(rows, n, k, False) > 0
    want = mxfp8.linear_mxfp8(x, w)
    monkeypatch.setattr(mxfp8, "_workspace_size", lambda *a: 0)
    assert torch.equal(mxfp8.linear_mxfp8(x, w), want)


@pytest.mark.parametrize("rows,n,k", [(64, 3584, 18944), (33, 4099, 12320), (77, 512, 8192)])
def test_captured_with_parts(dev, rows, n, k):
    """Graphs of products whose workgroups share k, two of them replayed in turn with other inputs between and
    at once on two streams: each has parts of its own."""
    from minimal_inference_amd import mxfp8

    assert mxfp8._workspace_size(rows, n, k, False) > 0
    sets = [(_whole(dev, rows, k, i), _whole(dev, n, k, 10 + i)) for i in range(2)]
    want = [mxfp8.linear_mxfp8(*s).clone() for s in sets]
    graphs = []
    for s in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = mxfp8.linear_mxfp8(*s)
        graphs.append((graph, out))
    for turn in range(6):
        for i in (turn % 2, 1 - turn % 2):
            graphs[i][1].fill_(7)
            graphs[i][0].replay()
            assert torch.equal(mxfp8.linear_mxfp8(*sets[1 - i]), want[1 - i])
            assert torch.equal(graphs[i][1], want[i])
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    for _, out in graphs:
        out.fill_(7)
    torch.cuda.synchronize(dev)
    for _ in range(8):
        for (graph, _), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize(dev)
    assert all(torch.equal(out, w) for (_, out), w in zip(graphs, want))


@pytest.mark.parametrize("rows,n,k", [(1, 64, 64), (20, 4864, 896), (64, 14336, 4096), (60, 18944, 512), (5, 18944, 416), (33, 41024, 96), (65, 96, 64), (300, 1120, 18944), (1030, 4096, 512),
                                      (2057, 8192, 1024), (4200, 2080, 1056)])
def test_gated_forms(dev, rows, n, k):
    """SiLU(gate) * up of exact products: bf16 by one rounding of fp32's value (2^-8, and 2^-20 for the exponential
    and the quotient), 8 bits by that value's codes but for values at a border."""
    from minimal_inference_amd.mxfp8 import linear_silu_mxfp8

    x, w = _whole(dev, rows, k, rows), _whole(dev, 2 * n, k, n)
    w.scales.sub_(9)  # (units of 2^-9: products around 1)
    both = (_values32(x) @ _values32(w).t()).double()
    want = both[:, :n] * torch.sigmoid(both[:, :n]) * both[:, n:]
    got = linear_silu_mxfp8(x, w).double()
    assert bool(((got - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -20) + 2.0 ** -133).all())
    m = linear_silu_mxfp8(x, w, quantize=True)
    unit = torch.exp2(m.scales.double() - 127.0).repeat_interleave(32, 1)
    # half a step of e4m3: 2^-4 of the value, 2^-10 of the unit below its least normal one
    assert bool(((om8.values(m.codes, m.scales).to(dev) - want).abs() <= (want.abs() * (2.0 ** -4 + 2.0 ** -20)).maximum(unit * 2.0 ** -10)).all())
    top = want.abs().view(rows, n // 32, 32).amax(-1)
    scale = torch.exp2(m.scales.double() - 127.0)
    assert bool((top * (1 - 2.0 ** -20) <= 448 * scale).all() and ((top * (1 + 2.0 ** -20) > 224 * scale) | (m.scales == 0)).all())


@pytest.mark.parametrize("exponent", [1, -1, -4, -8, -16, -100])
@pytest.mark.parametrize("rows", [3, 300])
def test_gate_alone(dev, rows, exponent):
    """Every code as a gate of a single product with an up of 1: silu within half a step of bf16 (2^-8 of the
    value, 2^-134 below its least normal one, which fp32's least, 2^-149, and its products' roundings may add to)."""
    from minimal_inference_amd.mxfp8 import MXFP8, linear_silu_mxfp8

    every = torch.arange(256, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
    every = every[every.float().isfinite()]
    n = every.numel()
    x, w = MXFP8(rows, 32, dev), MXFP8(2 * n, 32, dev)
    for m in (x, w):
        m.anchor.zero_()
        m.scales.fill_(127)
    x.codes[:, 0] = torch.linspace(0.1, 3.5, rows, device=dev).to(torch.float8_e4m3fn)
    x.codes[:, 1] = w.codes[n:, 1] = torch.ones((), device=dev).to(torch.float8_e4m3fn)
    w.codes[:n, 0] = every
    w.scales[:n] = 127 + exponent
    gate = x.codes[:, :1].double() * every.double() * 2.0 ** exponent
    want = gate * torch.sigmoid(gate)
    got = linear_silu_mxfp8(x, w).double()
    assert bool(((got - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -20) + 2.0 ** -134 + 2.0 ** -147).all())


def test_past_32_bits(dev):
    """Codes of x, of the matrix and an output past 2^32 bytes, rows at the far end."""
    from minimal_inference_amd.mxfp8 import MXFP8, linear_mxfp8

    k, rows = 1 << 16, (1 << 16) + 1024 + 40
    big = MXFP8(rows, k, dev)
    big.anchor.zero_()
    far = torch.cat((torch.arange(0, 40), torch.arange(rows - 40, rows))).to(dev)
    g = torch.Generator(device=dev).manual_seed(1)
    big.codes[far] = torch.randint(-3, 4, (80, k), device=dev, generator=g).float().to(torch.float8_e4m3fn)
    big.scales.fill_(127)
    small = _whole(dev, 48, k, 2)
    sv, fv = _values32(small), big.codes[far].float()
    want = fv @ sv.t()
    got = linear_mxfp8(big, small)  # rows past 32 bits, blocks of rows
    assert torch.equal(got[far], want.to(torch.bfloat16)) and not bool(got[40: rows - 40].any())
    got = linear_mxfp8(small, big)  # the matrix past them, few rows
    assert torch.equal(got[:, far], want.t().to(torch.bfloat16)) and not bool(got[:, 40: rows - 40].any())
    many = _whole(dev, 300, k, 3)
    got = linear_mxfp8(many, big)
    assert torch.equal(got[:, far], (_values32(many) @ fv.t()).to(torch.bfloat16))
    del big
    x, w = _whole(dev, 66000, 32, 4), _whole(dev, 36000, 32, 5)
    got = linear_mxfp8(x, w)  # 4.75 GB of output
    for at in (0, 32700, 65900):
        assert torch.equal(got[at: at + 100], (_values32(x)[at: at + 100] @ _values32(w).t()).to(torch.bfloat16))
