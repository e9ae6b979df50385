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


# (rows, n, k) that between them reach every form of the products, at widths of whole, half
# and odd 16-byte stores, k whole and in parts, and rows behind the last whole block
FORMS = [
    (512, 300, 160), (137, 384, 1024), (79, 50, 4128), (528, 36, 1184), (521, 96, 2048), (320, 77, 96), (263, 1836, 64),
    (1432, 34, 3680), (1290, 916, 7200), (649, 80, 6496), (288, 5555, 64), (591, 1676, 64), (265, 4096, 512),
    (1538, 385, 7424), (2179, 40, 5440), (648, 1936, 7808), (133, 11615, 64), (2568, 1588, 704), (528, 7352, 64),
    (1284, 2040, 3520), (2053, 467, 10080), (646, 1020, 8224), (1159, 1028, 7392), (650, 3891, 3392), (165, 10884, 64),
    (4100, 520, 96), (3596, 1060, 4064), (2307, 1688, 2752), (2621, 3078, 1056), (1205, 6524, 64), (2057, 4096, 160),
    (2563, 3116, 672), (1284, 4530, 64), (564, 8256, 64), (1295, 6303, 544), (771, 4957, 64), (1281, 5936, 64),
    (3360, 4820, 1088), (4127, 2019, 2080), (2305, 1744, 3776), (4139, 1968, 2144), (3355, 4800, 1088),
    (1411, 5808, 544), (2568, 3184, 672), (81, 1773, 7968), (1024, 2048, 256), (1923, 2064, 544)]


def _whole(rows, k, dev, g):
    """Whole numbers whose every sum over k is exact in fp32, with scales of 1 in 4 bits."""
    values = torch.tensor([0, 1, 2, 3, 4, 6, -1, -2, -3, -4, -6], device=dev, dtype=torch.float32)
    m = values[torch.randint(0, 11, (rows, k), device=dev, generator=g)]
    m[:, ::32] = torch.where(m[:, ::32] < 0, -6.0, 6.0)
    return m.to(torch.bfloat16)


def _both(x, weight, bias, n, silu, dev):
    """By the public entry and by the C entry without a workspace, into rows of wider buffers."""
    from minimal_inference_amd import _lib
    from minimal_inference_amd.mxfp4 import MXFP4, linear_mxfp4, linear_silu_mxfp4

    rows, k = x.shape
    out = torch.full((rows + 1, n + 8), 7.0, device=dev, dtype=torch.bfloat16)
    alone = torch.full_like(out, 7.0)
    if silu:
        linear_silu_mxfp4(x, weight, out=out[:rows, :n])
    else:
        linear_mxfp4(x, weight, bias, out=out[:rows, :n])
    ptr = (x.codes_ptr, 0, x.scales_ptr) if isinstance(x, MXFP4) else (x.data_ptr(), x.stride(0), None)
    _lib.call("mi_linear_mxfp4", *ptr, weight.codes_ptr, weight.scales_ptr, None if bias is None else bias.data_ptr(),
              alone.data_ptr(), alone.stride(0), rows, n, k, int(silu), None, 0, torch.cuda.current_stream().cuda_stream)
    for t in (out, alone):
        assert bool((t[rows] == 7).all()) and bool((t[:, n:] == 7).all())
    return out[:rows, :n], alone[:rows, :n]


@pytest.mark.parametrize("acts", ["bf16", "mxfp4"])
@pytest.mark.parametrize("rows,n,k", FORMS)
def test_a_bias_in_every_form(dev, rows, n, k, acts):
    """A whole number for each column, unlike its neighbours': the exact sums, rounded once."""
    from minimal_inference_amd.mxfp4 import quantize_mxfp4

    g = torch.Generator(device=dev).manual_seed(rows + n + k)
    x, w = _whole(rows, k, dev, g), _whole(n, k, dev, g)
    bias = ((torch.arange(n, device=dev) * 37) % 251 - 125).to(torch.bfloat16)
    assert 36 * k + 256 < 2 ** 24
    want = (x.float() @ w.float().t() + bias.float()).to(torch.bfloat16)
    for got in _both(quantize_mxfp4(x) if acts == "mxfp4" else x, quantize_mxfp4(w), bias, n, False, dev):
        assert torch.equal(got, want)


@pytest.mark.parametrize("silu", [False, True])
@pytest.mark.parametrize("acts", ["bf16", "mxfp4"])
@pytest.mark.parametrize("rows,n,k", FORMS)
def test_infinities_and_nan_in_every_form(dev, rows, n, k, acts, silu):
    """A NaN or an infinity in a row of x, the first and the last among them, and scale byte
    255 in a row of W reach that row or column alone; the rest is what it is without them."""
    from minimal_inference_amd.mxfp4 import MXFP4, quantize_mxfp4

    g = torch.Generator(device=dev).manual_seed(rows + n + k)
    x, w = _whole(rows, k, dev, g), _whole(2 * n if silu else n, k, dev, g)
    sums = x.float() @ w.float().t()  # (whole numbers below 2^24)
    x[0, k - 1], x[rows // 2, 0], x[rows // 2 + 1, k // 2], x[rows - 1, 33] = float("nan"), float("inf"), float("nan"), -float("inf")
    bad_rows = [0, rows // 2, rows // 2 + 1, rows - 1]
    codes, scales = quantize_mxfp4(w).to_codes()
    bad_cols = sorted({0, n // 2, n - 1})
    for i, c in enumerate(bad_cols):
        scales[c + (n if silu and i % 2 else 0), [0, -1, k // 64][i]] = 255
    weight = MXFP4.from_codes(codes, scales)
    xx = quantize_mxfp4(x) if acts == "mxfp4" else torch.cat([x, torch.full_like(x[:, :32], float("nan"))], 1)[:, :k]
    reached = torch.zeros(rows, n, dtype=torch.bool, device=dev)
    reached[bad_rows] = True
    reached[:, bad_cols] = True
    if silu:
        gate, up = sums.double().chunk(2, -1)
        ref = gate * torch.sigmoid(gate) * up
    for got in _both(xx, weight, None, n, silu, dev):
        assert torch.equal(got.isfinite(), ~reached)
        assert bool(got[:, bad_cols].isnan().all())
        if silu:  # fp32: the exponential, the quotient and the products round 8 times
            near = (got.double() - ref).abs() <= (2 ** -8 + 8 * 2 ** -24) * ref.abs() + 1e-30
            assert bool((near | reached).all())
        else:
            assert bool(((got == sums.to(torch.bfloat16)) | reached).all())
