"""GPU: the gated products' fp32 sums at widths that fill no tile, and past 32 bits of offset.

Bars: an 8-bit product's is that of test_gpu_mxfp8 (2^-10 of the 2-norm of its products).  With 4-bit weights and bf16 rows
products are exact in fp32 and their sum loses 2^-24 an addition at most, k of them in the worst order.
"""

from __future__ import annotations

import pytest
import torch

from oracle import mxfp8 as om8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [4, 36, 100, 260, 900])
@pytest.mark.parametrize("rows,k", [(1, 96), (20, 1056), (64, 4864), (65, 96), (200, 8192), (300, 160), (520, 1056)])
def test_sums_of_ragged_widths(dev, rows, k, n):
    from minimal_inference_amd.mxfp4 import gate_up_mxfp4, quantize_mxfp4
    from minimal_inference_amd.mxfp8 import gate_up_mxfp8, quantize_mxfp8

    g = torch.Generator(device=dev).manual_seed(rows + n + k)
    x = torch.randn(rows, k, device=dev, generator=g).to(torch.bfloat16)
    w = torch.randn(2 * n, k, device=dev, generator=g).to(torch.bfloat16)
    room = torch.full((rows + 2, 2 * n + 8), 7.0, device=dev)

    def whole(call):
        room.fill_(7.0)
        out = room[1: rows + 1, 4: 4 + 2 * n]
        assert call(out) is out
        assert bool((room[0] == 7).all() and (room[-1] == 7).all() and (room[:, :4] == 7).all() and (room[:, 4 + 2 * n:] == 7).all())
        return out.double()

    m, w8 = quantize_mxfp8(x), quantize_mxfp8(w)
    vx, vw = om8.values(m.codes, m.scales).to(dev), om8.values(w8.codes, w8.scales).to(dev)
    got = whole(lambda out: gate_up_mxfp8(m, w8, out))
    assert bool(((got - vx @ vw.t()).abs() <= 2.0 ** -10 * (vx.square() @ vw.square().t()).sqrt()).all())
    w4 = quantize_mxfp4(w)
    v4 = w4.dequantize().double()
    got = whole(lambda out: gate_up_mxfp4(x, w4, out))
    assert bool(((got - x.double() @ v4.t()).abs() <= k * 2.0 ** -24 * (x.double().abs() @ v4.abs().t())).all())


def test_rows_past_32_bits(dev):
    """More than 2^31 sums: the last rows' and their adapters' are those of a call of these rows alone."""
    from minimal_inference_amd.adapters import AdapterPlan, Adapters, add_adapters_silu
    from minimal_inference_amd.mxfp8 import gate_up_mxfp8, linear_silu_mxfp8, quantize_mxfp8

    rows, k, half, last = 76800, 64, 14336, 512
    g = torch.Generator(device=dev).manual_seed(3)
    randn = lambda *s: torch.randn(*s, device=dev, generator=g).to(torch.bfloat16)  # noqa: E731
    x, w = randn(rows, k), quantize_mxfp8(randn(2 * half, k))
    ad = Adapters(randn(2, 16, k), randn(2, 2 * half, 8), torch.ones(2, device=dev), [half, half])
    slot = (torch.arange(rows, device=dev) % 3 - 1).to(torch.int32)
    plan, own = AdapterPlan(rows, 2, dev), AdapterPlan(last, 2, dev)
    plan.plan(slot)
    own.plan(slot[-last:].contiguous())
    m, tail = quantize_mxfp8(x), quantize_mxfp8(x[-last:])
    y = gate_up_mxfp8(m, w)
    assert y.numel() > 1 << 31
    # (forms may differ in their order of sums: one group of 64 products here, whose order is the instruction's)
    assert torch.equal(y[-last:], gate_up_mxfp8(tail, w))
    q = add_adapters_silu(y, m, ad, plan, quantize=True)
    base = linear_silu_mxfp8(tail, w, quantize=True)
    none = slot[-last:] < 0
    assert torch.equal(q.codes.view(torch.uint8)[-last:][none], base.codes.view(torch.uint8)[none])
    assert torch.equal(q.scales[-last:][none], base.scales[none])
    alone = add_adapters_silu(y[-last:].clone(), tail, ad, own, quantize=True)
    # (A x in parts as the number of rows asks for: within a step of e4m3 each)
    a, b = om8.values(q.codes[-last:], q.scales[-last:]), om8.values(alone.codes, alone.scales)
    unit = torch.exp2(torch.maximum(q.scales[-last:], alone.scales).double() - 127).repeat_interleave(32, 1)
    assert bool(((a - b).abs() <= (a.abs().maximum(b.abs()) * 2.0 ** -3).maximum(unit * 2.0 ** -9)).all())
