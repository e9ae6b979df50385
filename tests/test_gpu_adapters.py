"""GPU: adapters of many requests against the 64-bit sum.

Bars.  v = A x is a sum of k exact products in fp32: within 4 sqrt(k) 2^-24 of the sum of their
magnitudes.  It enters the second product as two bf16 numbers, 2^-16 of it off at most, and scale * v
is rounded once (2^-24).  The second sum is of rank such products, y is added (fp32), and
the result rounded once to bf16 (2^-8).
"""

from __future__ import annotations

import pytest
import torch

from oracle import mxfp8 as om8

pytestmark = pytest.mark.gpu


def _make(dev, rows, k, pieces, rank, slots, seed=0, x8=False):
    from minimal_inference_amd.adapters import Adapters
    from minimal_inference_amd.mxfp8 import quantize_mxfp8

    g = torch.Generator(device=dev).manual_seed(seed + rows + k)

    def randn(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    n = sum(pieces)
    x = randn(rows, k).to(torch.bfloat16)
    ad = Adapters((randn(slots, len(pieces) * rank, k) * k ** -0.5).to(torch.bfloat16),
                  randn(slots, n, rank).to(torch.bfloat16), 0.25 + torch.rand(slots, device=dev, generator=g), pieces)
    slot = torch.randint(-1, slots, (rows,), device=dev, generator=g).to(torch.int32)
    y = randn(rows, n).to(torch.bfloat16)
    values = x.double()
    if x8:
        x = quantize_mxfp8(x)
        values = om8.values(x.codes, x.scales)
    return x, values, ad, slot, y


def _want(values, ad, slot, y):
    """The sum and how far a result may be from it, row by row's adapter."""
    ref, tol = y.double().clone(), torch.zeros_like(y, dtype=torch.float64)
    k, rank = ad.k, ad.rank
    for s in range(ad.slots):
        mine = (slot == s).nonzero()[:, 0]
        a, b, scale = ad.a[s].double(), ad.b[s].double(), ad.scale[s].double()
        v = values[mine] @ a.t() * scale
        ev = 4 * k ** 0.5 * 2.0 ** -24 * (values[mine].abs() @ a.abs().t()) * scale + (2.0 ** -16 + 2.0 ** -24) * v.abs()
        first = 0
        for i, n in enumerate(ad.pieces):
            part, w = slice(i * rank, (i + 1) * rank), b[first: first + n]
            ref[mine, first: first + n] += v[:, part] @ w.t()
            tol[mine, first: first + n] += ev[:, part] @ w.abs().t() + (rank + 2) * 2.0 ** -24 * (v[:, part].abs() @ w.abs().t())
            first += n
    tol += 2.0 ** -24 * y.double().abs()
    return ref, tol + 2 ** -8 * (ref.abs() + tol)


@pytest.mark.parametrize("x8", [False, True])
@pytest.mark.parametrize("k,pieces,rank", [(32, [16], 8), (96, [48, 16], 16), (896, [896, 128, 128], 16), (1056, [304], 24),
                                           (544, [64, 32, 16], 64), (4864, [896], 32), (256, [160, 160], 128),
                                           (1056, [9728], 32), (896, [4864, 4864], 16),
                                           (160, [16] * 8, 8)])
@pytest.mark.parametrize("rows,slots", [(1, 1), (3, 5), (17, 2), (64, 1), (130, 7), (300, 40), (320, 3), (321, 3), (512, 3), (513, 3), (1000, 1),
                                        (900, 30)])
def test_add_adapters(dev, rows, slots, k, pieces, rank, x8):
    """Odd numbers of rows and adapters, rows without one among them; in place and into an out, whose
    surroundings stay; strided rows."""
    from minimal_inference_amd.adapters import AdapterPlan, add_adapters

    x, values, ad, slot, y = _make(dev, rows, k, pieces, rank, slots, x8=x8)
    plan = AdapterPlan(rows + 3, slots, dev)
    plan.plan(slot)
    ref, tol = _want(values, ad, slot, y)
    n = sum(pieces)
    room = torch.full((rows, n + 24), 7.0, device=dev, dtype=torch.bfloat16)
    before = y.clone()
    got = add_adapters(y, x, ad, plan, out=room[:, 8: 8 + n])
    assert torch.equal(y, before)
    assert bool(((got.double() - ref).abs() <= tol).all())
    assert torch.equal(got[slot < 0], y[slot < 0])
    assert bool((room[:, :8] == 7).all()) and bool((room[:, 8 + n:] == 7).all())
    wide = torch.zeros(rows, n + 40, device=dev, dtype=torch.bfloat16)
    wide[:, 16: 16 + n] = y
    assert add_adapters(wide[:, 16: 16 + n], x, ad, plan).data_ptr() == wide[:, 16:].data_ptr()
    assert torch.equal(wide[:, 16: 16 + n], got)
    assert not bool(wide[:, :16].any()) and not bool(wide[:, 16 + n:].any())


def test_plan_lists_every_row_once(dev):
    """Ids outside the adapters are none; no rows, one, more than the plan's threads, all of one adapter,
    the most adapters; the tiles hold each row once under its adapter."""
    from minimal_inference_amd.adapters import AdapterPlan

    for rows, slots, how in ((0, 3, "mixed"), (1, 1, "mixed"), (5, 1023, "mixed"), (4097, 1023, "mixed"), (5000, 3, "runs"),
                             (2048, 4, "one"), (3001, 2, "wild"), (100, 7, "none")):
        g = torch.Generator().manual_seed(rows)
        slot = torch.randint(-1, slots, (rows,), generator=g)
        if how == "runs":
            slot = slot.sort()[0]
        if how == "one":
            slot[:] = 2
        if how == "none":
            slot[:] = -1
        if how == "wild":
            slot = torch.randint(-(1 << 31), 1 << 31, (rows,), generator=g)
            slot[::3] = 1
        slot = slot.to(torch.int32)
        plan = AdapterPlan(rows, slots, dev)
        plan.plan(slot.to(dev))
        words = plan.buffer.view(torch.int32).cpu()
        if rows == 0:
            assert int(words[0]) == 0
            continue
        height = 16 if rows <= 320 else 64
        most = min(rows, slots + 1) + rows // height
        assert 0 < int(words[0]) <= most and words[1:3].tolist() == [rows, slots]
        lists = words[4: 4 + most * height].view(most, height)
        seen = []
        for i, (s, count) in enumerate(words[4 + most * height:][: 2 * int(words[0])].view(-1, 2).tolist()):
            assert 0 < count <= height
            seen.append(lists[i, :count])
            mine = slot[seen[-1].long()]
            own = (mine == s) if s >= 0 else (mine < 0) | (mine >= slots)
            assert bool(own.all())
        assert torch.equal(torch.cat(seen).sort()[0], torch.arange(rows, dtype=torch.int32))


def test_a_row_depends_on_no_other(dev):
    """The same rows in another order, and beside rows of infinities and NaN, give the same bits."""
    from minimal_inference_amd.adapters import AdapterPlan, add_adapters

    x, _, ad, slot, y = _make(dev, 200, 256, [96, 32], 16, 3)
    plan = AdapterPlan(400, 3, dev)
    plan.plan(slot)
    want = add_adapters(y, x, ad, plan, out=torch.empty_like(y))
    order = torch.randperm(200, device=dev, generator=torch.Generator(device=dev).manual_seed(1))
    plan.plan(slot[order].contiguous())
    assert torch.equal(add_adapters(y[order], x[order], ad, plan), want[order])
    x2, y2 = x.clone(), y.clone()
    x2[::2], y2[1::4] = float("nan"), float("inf")
    x2[2::4] = float("inf")
    plan.plan(slot)
    got = add_adapters(y2, x2, ad, plan)
    assert torch.equal(got[3::4], want[3::4])


def test_set_and_clear(dev):
    from minimal_inference_amd.adapters import AdapterPlan, Adapters, add_adapters

    g = torch.Generator(device=dev).manual_seed(5)
    ad = Adapters.empty(3, 64, [32, 16], 24, dev)
    a0, b0 = torch.randn(8, 64, device=dev, generator=g), torch.randn(32, 8, device=dev, generator=g)
    a1, b1 = torch.randn(5, 64, device=dev, generator=g), torch.randn(16, 5, device=dev, generator=g)
    ad.set(1, [(a0, b0), (a1, b1)], 0.5)
    ad.set(2, [None, (a1, b1)], 2.0)
    x = torch.randn(6, 64, device=dev, generator=g).to(torch.bfloat16)
    y = torch.zeros(6, 48, device=dev, dtype=torch.bfloat16)
    slot = torch.tensor([0, 1, 2, -1, 1, 2], device=dev, dtype=torch.int32)
    plan = AdapterPlan(6, 3, dev)
    plan.plan(slot)
    got = add_adapters(y, x, ad, plan, out=torch.empty_like(y))
    bf = lambda t: t.to(torch.bfloat16).double()  # noqa: E731
    first, second = x.double() @ bf(a0).t() @ bf(b0).t(), x.double() @ bf(a1).t() @ bf(b1).t()
    want = torch.zeros(6, 48, dtype=torch.float64, device=dev)
    for i in (1, 4):
        want[i] = 0.5 * torch.cat([first[i], second[i]])
    for i in (2, 5):
        want[i, 32:] = 2.0 * second[i]
    ref, tol = _want(x.double(), ad, slot, y)
    assert float((ref - want).abs().max()) < 1e-9
    assert bool(((got.double() - want).abs() <= tol).all())
    ad.clear(1)
    assert not bool(add_adapters(y, x, ad, plan, out=torch.empty_like(y))[[1, 4]].any())


@pytest.mark.parametrize("x8", [False, True])
@pytest.mark.parametrize("k,half,rank", [(32, 16, 8), (96, 32, 16), (896, 4864, 16), (1056, 304, 24), (544, 1184, 64), (256, 160, 128), (544, 9728, 32)])
@pytest.mark.parametrize("rows,slots", [(1, 1), (3, 5), (17, 2), (130, 7), (320, 3), (321, 3), (900, 30)])
def test_add_adapters_silu(dev, rows, slots, k, half, rank, x8):
    """SiLU(gate) * up of the sums: gate and up within their bars dg and du of the 64-bit sums G and U (without
    the rounding to bf16), silu's slope is 1.1 at most and its value |G| at most, so the product is within
    1.1 dg (|U| + du) + |G| du + 2^-20 of itself, and rounded once: bf16 2^-8, or e4m3 2^-4 (2^-10 of the block's
    unit below its least normal code). y stays, and what lies around out."""
    from minimal_inference_amd.adapters import AdapterPlan, add_adapters_silu

    x, values, ad, slot, y = _make(dev, rows, k, [half, half], rank, slots, x8=x8)
    plan = AdapterPlan(rows, slots, dev)
    plan.plan(slot)
    ref, tol = _want(values, ad, slot, y)
    tol = (tol - 2 ** -8 * ref.abs()) / (1 + 2 ** -8) + 2.0 ** -24 * ref.abs()  # (the bar before the rounding; the sum's own)
    G, U, dg, du = ref[:, :half], ref[:, half:], tol[:, :half], tol[:, half:]
    want = G * torch.sigmoid(G) * U
    near = 1.1 * dg * (U.abs() + du) + G.abs() * du + 2.0 ** -20 * want.abs()
    y0 = y.clone()
    room = torch.full((rows + 2, half + 8), 7.0, dtype=torch.bfloat16, device=dev)
    out = add_adapters_silu(y, x, ad, plan, out=room[1: rows + 1, :half])
    assert bool(((out.double() - want).abs() <= near + 2 ** -8 * (want.abs() + near)).all())
    assert bool((room[0] == 7).all() and (room[-1] == 7).all() and (room[:, half:] == 7).all())
    assert torch.equal(add_adapters_silu(y, x, ad, plan), out)
    if half % 32 == 0:
        m = add_adapters_silu(y, x, ad, plan, quantize=True)
        unit = torch.exp2(m.scales.double() - 127.0).repeat_interleave(32, 1)
        got = om8.values(m.codes, m.scales).to(dev)
        assert bool(((got - want).abs() <= near + ((want.abs() + near) * 2.0 ** -4).maximum(unit * 2.0 ** -10)).all())
        top, slack = want.abs().view(rows, half // 32, 32).amax(-1), near.view(rows, half // 32, 32).amax(-1)
        scale = torch.exp2(m.scales.double() - 127.0)
        assert bool((top - slack <= 448 * scale).all() and ((top + slack > 224 * scale) | (m.scales == 0)).all())
    else:
        with pytest.raises(ValueError):
            add_adapters_silu(y, x, ad, plan, quantize=True)
    assert torch.equal(y, y0)


def test_add_adapters_silu_refuses(dev):
    from minimal_inference_amd.adapters import AdapterPlan, add_adapters_silu
    from minimal_inference_amd.mxfp8 import MXFP8

    x, _, ad, slot, y = _make(dev, 5, 64, [32, 32], 8, 2)
    plan = AdapterPlan(5, 2, dev)
    plan.plan(slot)
    for bad in (y, y[:, :32], torch.empty(5, 64, dtype=torch.bfloat16, device=dev), torch.empty(4, 32, dtype=torch.bfloat16, device=dev)):
        with pytest.raises(ValueError):
            add_adapters_silu(y, x, ad, plan, out=bad)
    for bad in (MXFP8(5, 64, dev), y[:, :32]):
        with pytest.raises(ValueError):
            add_adapters_silu(y, x, ad, plan, out=bad, quantize=True)
    _, _, other, _, _ = _make(dev, 5, 64, [48, 16], 8, 2)
    with pytest.raises(ValueError, match="gate and up"):
        add_adapters_silu(y, x, other, plan)


def test_add_adapters_silu_replayed_after_another_batch(dev):
    """NaN in bf16 and in 8 bits after a plan of another number of rows; its own bits again after its own."""
    from minimal_inference_amd.adapters import AdapterPlan, add_adapters_silu

    x, _, ad, slot, y = _make(dev, 40, 64, [96, 96], 8, 2)
    plan = AdapterPlan(40, 2, dev)
    plan.plan(slot)
    want = [add_adapters_silu(y, x, ad, plan), add_adapters_silu(y, x, ad, plan, quantize=True)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [add_adapters_silu(y, x, ad, plan), add_adapters_silu(y, x, ad, plan, quantize=True)]
    for _ in range(3):
        plan.plan(slot[:33])
        graph.replay()
        assert bool(got[0].isnan().all() and (got[1].scales == 255).all()) and not bool(got[1].codes.view(torch.uint8).any())
        plan.plan(slot)
        graph.replay()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1].scales, want[1].scales)
        assert torch.equal(got[1].codes.view(torch.uint8), want[1].codes.view(torch.uint8))
