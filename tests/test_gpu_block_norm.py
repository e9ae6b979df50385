"""GPU: the norms after a block and before the next, against the formula in 64 bits.

Bars.  x_out: one bf16 rounding (2^-8 relative) of s, which fp32 holds to 16 roundings of
its terms.  h: one rounding of s * rsqrt(..) * w, whose factors fp32 holds to 32
roundings; the sums of squares are of like signs, so their relative error is no more
than the tree's depth, which those counts cover.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _reference(x, y, post, pre, gate, scale, eps):
    x, y = x.double(), y.double()
    z = scale * y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps) * post.double()
    if gate is not None:
        z = z * gate.double()
    s = x + z
    h = s * torch.rsqrt(s.square().mean(-1, keepdim=True) + eps) * pre.double()
    far_s = 16 * U * (x.abs() + z.abs())
    far_h = torch.rsqrt(s.square().mean(-1, keepdim=True) + eps) * pre.double().abs() * far_s + 32 * U * h.abs()
    return s, h, far_s, far_h


def _inputs(rows, hidden, gate, dev):
    g = torch.Generator(device=dev).manual_seed(rows * 131 + hidden)

    def randn(*shape):
        return torch.randn(*shape, device=dev, generator=g).to(torch.bfloat16)

    shape = {"none": None, "channel": (hidden,), "token": (rows, 1), "full": (rows, hidden)}[gate]
    return 3 * randn(rows, hidden), randn(rows, hidden), 1 + randn(hidden) / 8, 1 + randn(hidden) / 8, \
        None if shape is None else randn(*shape)


@pytest.mark.parametrize("gate", ["none", "channel", "token", "full"])
@pytest.mark.parametrize("hidden", [8, 64, 104, 512, 520, 896, 3584, 4096, 8192, 8200, 16384])
@pytest.mark.parametrize("rows", [1, 2, 7, 130])
def test_post_norm_add_rms_norm(dev, rows, hidden, gate):
    from minimal_inference_amd.dense import post_norm_add_rms_norm

    x, y, post, pre, gt = _inputs(rows, hidden, gate, dev)
    s, h, far_s, far_h = _reference(x, y, post, pre, gt, 0.25, 1e-6)
    x0, out = x.clone(), torch.empty_like(x)
    got = post_norm_add_rms_norm(x, y, post, pre, 1e-6, gate=gt, scale=0.25, x_out=out)
    assert torch.equal(x, x0)
    assert bool(((out.double() - s).abs() <= 2 ** -8 * s.abs() + far_s).all())
    assert bool(((got.double() - h).abs() <= 2 ** -8 * h.abs() + far_h).all())
    again = post_norm_add_rms_norm(x, y, post, pre, 1e-6, gate=gt, scale=0.25, h_out=y)  # in place, h over y
    assert torch.equal(x, out) and torch.equal(again, got) and again.data_ptr() == y.data_ptr()


def test_strides_and_what_lies_around(dev):
    """Rows of wider buffers on every side, a strided gate of either kind."""
    from minimal_inference_amd.dense import post_norm_add_rms_norm

    rows, hidden = 9, 256
    x, y, post, pre, full = _inputs(rows, hidden, "full", dev)
    wide = lambda t: torch.cat([t, torch.full_like(t, 7.0)], 1)[:, :hidden]  # noqa: E731
    for gt in (full, full[:, 3:4]):
        want_x = torch.empty_like(x)
        want = post_norm_add_rms_norm(x, y, post, pre, 1e-5, gate=gt.contiguous(), x_out=want_x)
        xb, hb = torch.full((rows + 1, hidden + 16), 7.0, device=dev, dtype=torch.bfloat16), \
            torch.full((rows + 1, hidden + 8), 7.0, device=dev, dtype=torch.bfloat16)
        got = post_norm_add_rms_norm(wide(x), wide(y), post, pre, 1e-5, gate=wide(gt) if gt is full else gt,
                                     x_out=xb[:rows, 8:8 + hidden], h_out=hb[:rows, :hidden])
        assert torch.equal(got, want) and torch.equal(xb[:rows, 8:8 + hidden], want_x)
        assert bool((xb[rows] == 7).all()) and bool((xb[:, :8] == 7).all()) and bool((xb[:, -8:] == 7).all())
        assert bool((hb[rows] == 7).all()) and bool((hb[:, hidden:] == 7).all())


def test_zero_rows_infinities_and_defaults(dev):
    """Zero rows stay zero (eps keeps the norms finite); an infinity or a NaN stays in
    its row; scale 1 and no gate by default; no rows."""
    from minimal_inference_amd.dense import post_norm_add_rms_norm

    x, y, post, pre, _ = _inputs(6, 512, "none", dev)
    x[0], y[0], y[1] = 0, 0, 0
    y[3, 5], x[4, 0] = float("inf"), float("nan")
    want_s, want_h, far_s, far_h = _reference(x, y, post, pre, None, 1.0, 1e-6)
    h = post_norm_add_rms_norm(x, y, post, pre, 1e-6)
    assert bool((x[0] == 0).all()) and bool((h[0] == 0).all())
    keep = [0, 1, 2, 5]
    assert bool(((x - want_s).abs() <= 2 ** -8 * want_s.abs() + far_s)[keep].all())
    assert bool(((h - want_h).abs() <= 2 ** -8 * want_h.abs() + far_h)[keep].all())
    assert bool(x[3, 5].isnan()) and bool(h[3].isnan().any()) and bool(h[4].isnan().all())
    assert post_norm_add_rms_norm(x[:0], y[:0], post, pre, 1e-6).shape == (0, 512)


def test_one_row_of_any_stride(dev):
    from minimal_inference_amd.dense import post_norm_add_rms_norm

    x, y, post, pre, gate = _inputs(1, 64, "full", dev)
    want_x, odd_x = torch.empty_like(x), torch.empty_like(x)
    want = post_norm_add_rms_norm(x, y, post, pre, 1e-6, gate=gate, x_out=want_x)
    odd = lambda t: t.as_strided((1, 64), (5, 1))  # noqa: E731
    assert torch.equal(post_norm_add_rms_norm(odd(x), odd(y), post, pre, 1e-6, gate=odd(gate), x_out=odd(odd_x)), want)
    assert torch.equal(odd_x, want_x)


def test_refused(dev):
    from minimal_inference_amd.dense import post_norm_add_rms_norm

    x, y, post, pre, gate = _inputs(4, 64, "full", dev)
    for a, kw in [((x, y[:3], post, pre), {}), ((x, y[:, :56], post, pre), {}), ((x.float(), y, post, pre), {}),
                  ((x, y, post[:32], pre), {}), ((x, y, post, pre), {"gate": gate[:, :8]}),
                  ((x, y, post, pre), {"gate": gate.float()}), ((x, y, post, pre), {"x_out": x[:2]}),
                  ((x, y, post, pre), {"h_out": y[:, ::2]}), ((x[:, :60], y[:, :60], post[:60], pre[:60]), {}),
                  ((x.cpu(), y, post, pre), {}), ((x, y, post.clone().requires_grad_(), pre), {}),
                  ((x[:, 4:], y[:, 4:], post[4:], pre[4:]), {}), ((x[:1].expand(4, 64), y, post, pre), {}),
                  ((x, y, post, pre), {"h_out": y[:1].expand(4, 64)})]:
        with pytest.raises(ValueError):
            post_norm_add_rms_norm(*a, 1e-6, **kw)


def test_replayed(dev):
    from minimal_inference_amd.dense import post_norm_add_rms_norm

    x, y, post, pre, gate = _inputs(5, 896, "token", dev)
    out = torch.empty_like(x)
    post_norm_add_rms_norm(x, y, post, pre, 1e-6, gate=gate, x_out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h = post_norm_add_rms_norm(x, y, post, pre, 1e-6, gate=gate, x_out=out)
    for seed in range(3):
        x.copy_(torch.randn(5, 896, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        held = (out.clone(), h.clone())
        want = torch.empty_like(x)
        assert torch.equal(post_norm_add_rms_norm(x, y, post, pre, 1e-6, gate=gate, x_out=want), held[1])
        assert torch.equal(want, held[0])
