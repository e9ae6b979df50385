"""GPU: what the operators over 4-bit matrices and the norms around a block refuse, and
their largest forms with a bias, infinities and NaN."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_tangents_are_refused(dev):
    """A forward-mode tangent would be dropped: it is refused like a gradient, on every
    argument; tensors without one pass inside a level, and after it all do."""
    from torch.autograd import forward_ad

    from minimal_inference_amd.dense import post_norm_add_rms_norm
    from minimal_inference_amd.mxfp4 import linear_mxfp4, linear_silu_mxfp4, quantize_mxfp4

    x = torch.randn(4, 64, device=dev).to(torch.bfloat16)
    w = quantize_mxfp4(torch.randn(32, 64, device=dev).to(torch.bfloat16))
    bias, norm = torch.ones(32, device=dev, dtype=torch.bfloat16), torch.ones(64, device=dev, dtype=torch.bfloat16)
    want = linear_mxfp4(x, w, bias), linear_silu_mxfp4(x, w), quantize_mxfp4(x).dequantize()
    norms = post_norm_add_rms_norm(x, x, norm, norm, 1e-6, gate=norm, x_out=torch.empty_like(x))
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        out = dual(torch.empty_like(want[0]))
        for bad in [lambda: linear_mxfp4(dual(x), w), lambda: linear_mxfp4(x, w, dual(bias)),
                    lambda: linear_mxfp4(x, w, out=out), lambda: linear_silu_mxfp4(dual(x), w),
                    lambda: quantize_mxfp4(dual(x)), lambda: w.dequantize(dual(torch.empty(32, 64, device=dev, dtype=x.dtype))),
                    lambda: post_norm_add_rms_norm(dual(x), x, norm, norm, 1e-6, x_out=torch.empty_like(x)),
                    lambda: post_norm_add_rms_norm(x, dual(x), norm, norm, 1e-6, x_out=torch.empty_like(x)),
                    lambda: post_norm_add_rms_norm(x, x, dual(norm), norm, 1e-6, x_out=torch.empty_like(x)),
                    lambda: post_norm_add_rms_norm(x, x, norm, dual(norm), 1e-6, x_out=torch.empty_like(x)),
                    lambda: post_norm_add_rms_norm(x, x, norm, norm, 1e-6, gate=dual(norm), x_out=torch.empty_like(x)),
                    lambda: post_norm_add_rms_norm(x, x, norm, norm, 1e-6, x_out=dual(torch.empty_like(x))),
                    lambda: post_norm_add_rms_norm(x, x, norm, norm, 1e-6, x_out=torch.empty_like(x), h_out=dual(x.clone()))]:
            with pytest.raises(ValueError, match="tangent"):
                bad()
        assert torch.equal(linear_mxfp4(x, w, bias), want[0])
        with torch.inference_mode():  # (no derivatives are asked for there)
            assert torch.equal(linear_silu_mxfp4(dual(x), w), want[1])
        x2 = dual(x)
    assert torch.equal(quantize_mxfp4(x2).dequantize(), want[2])
    assert torch.equal(post_norm_add_rms_norm(x, x, norm, norm, 1e-6, gate=norm, x_out=torch.empty_like(x)), norms)


def test_widths_past_32_bits_are_refused(dev):
    """Sizes whose lower 32 bits are a width that the kernels take."""
    from minimal_inference_amd.dense import post_norm_add_rms_norm
    from minimal_inference_amd.sampling import Sampler

    wide = torch.empty(1, (1 << 32) + 64, device=dev, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="hidden"):
        post_norm_add_rms_norm(wide, wide, wide[0], wide[0], 1e-6, h_out=wide)
    s = Sampler(dev, 1, vocab=64)
    s.set_params([1.0])
    with pytest.raises(ValueError, match="tokens"):
        s.draw(wide, torch.zeros(1, device=dev))


@pytest.mark.parametrize("acts", ["bf16", "mxfp4"])
@pytest.mark.parametrize("rows", [1, 20, 200])
def test_linear_into_the_columns_beside_x(dev, rows, acts):
    """x, out and the bias in one buffer, columns and rows apart: as with tensors of their own."""
    from minimal_inference_amd.mxfp4 import linear_mxfp4, quantize_mxfp4

    n, k = 96, 160
    w = quantize_mxfp4(torch.randn(n, k, device=dev).to(torch.bfloat16))
    buffer = torch.randn(rows + 1, k + n + 8, device=dev).to(torch.bfloat16)
    x, out, bias = buffer[:rows, :k], buffer[:rows, k:k + n], buffer[rows, :n]
    xx = quantize_mxfp4(x) if acts == "mxfp4" else x
    want = linear_mxfp4(xx, w, bias.clone())
    around = buffer.clone()
    assert linear_mxfp4(xx, w, bias, out=out).data_ptr() == out.data_ptr()
    around[:rows, k:k + n] = want
    assert torch.equal(buffer, around)
    for bad in (buffer[:rows, k - 1:k - 1 + n], buffer[1:rows + 1, :n], buffer[rows:, :n].expand(rows, n)):
        if acts == "bf16" or bad.data_ptr() == bias.data_ptr():
            with pytest.raises(ValueError):
                linear_mxfp4(xx, w, bias, out=bad)


@pytest.mark.parametrize("rows", [1, 7, 300])
def test_norms_in_place_of_any_input(dev, rows):
    """Outputs over x, y or a full gate, over a column of a wider buffer and beside x in one:
    the bits of a call with tensors of their own; overlaps between rows are refused."""
    from minimal_inference_amd.dense import post_norm_add_rms_norm

    hidden = 264
    randn = lambda *s: torch.randn(*s, device=dev).to(torch.bfloat16)  # noqa: E731
    x, y, gate, post, pre = randn(rows, hidden), randn(rows, hidden), randn(rows, hidden), randn(hidden), randn(hidden)
    want_x = torch.empty_like(x)
    want = post_norm_add_rms_norm(x, y, post, pre, 1e-6, gate=gate, x_out=want_x)
    for xo, ho in (("x", "y"), ("y", "x"), ("gate", "x"), ("x", "gate"), ("beside", "x"), ("y", "beside")):
        wide = randn(rows, 2 * hidden + 8)
        wide[:, :hidden] = x
        at = {"x": wide[:, :hidden], "y": y.clone(), "gate": gate.clone(), "beside": wide[:, hidden:2 * hidden]}
        got = post_norm_add_rms_norm(at["x"], at["y"], post, pre, 1e-6, gate=at["gate"], x_out=at[xo], h_out=at[ho])
        assert got is at[ho] and torch.equal(got, want) and torch.equal(at[xo], want_x)
    buffer = randn(rows + 1, hidden)
    buffer[:rows] = x
    for bad in [dict(x_out=buffer[:rows], h_out=buffer[:rows])] + ([dict(x_out=buffer[1:]), dict(h_out=buffer[1:])] if rows > 1 else []):
        with pytest.raises(ValueError, match="overlaps"):
            post_norm_add_rms_norm(buffer[:rows], y, post, pre, 1e-6, **bad)
    with pytest.raises(ValueError, match="overlaps"):
        post_norm_add_rms_norm(x, y, post, buffer[rows], 1e-6, x_out=buffer[1:])
    with pytest.raises(ValueError, match="overlaps"):
        post_norm_add_rms_norm(x, x, post, pre, 1e-6, h_out=x)
