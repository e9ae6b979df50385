"""GPU: MXFP4 matrices and the linear layers over them against 64-bit restatements.

Bars.  Quantisation, packing and the return to bf16 are exact.  A product's sum of k
exact products in fp32 stays within 4 sqrt(k) 2^-24 sum |x w| of the exact one
(independent rounding errors) and is rounded once to bf16 (2^-8 relative).
"""

from __future__ import annotations

import pytest
import torch

from oracle import mxfp4 as omx

pytestmark = pytest.mark.gpu


def _normals(rows, cols, dev, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn(rows, cols, device=dev, generator=g)
    return (x * torch.exp(2 * torch.randn(rows, 1, device=dev, generator=g))).to(torch.bfloat16)


def _weight(n, k, dev, seed):
    """Codes and scale bytes of a random matrix, its MXFP4 form and its values (64 bits, on the GPU)."""
    from minimal_inference_amd.mxfp4 import MXFP4

    g = torch.Generator(device=dev).manual_seed(seed)
    codes = torch.randint(0, 256, (n, k // 2), device=dev, generator=g, dtype=torch.uint8)
    scales = torch.randint(118, 124, (n, k // 32), device=dev, generator=g, dtype=torch.uint8)
    grid = torch.tensor(omx.GRID + tuple(-v for v in omx.GRID), dtype=torch.float64, device=dev)
    code = torch.stack((codes & 15, codes >> 4), -1).view(n, k // 32, 32).long()
    values = (grid[code] * torch.exp2(scales.double() - 127)[..., None]).view(n, k)
    return codes, scales, MXFP4.from_codes(codes, scales), values


@pytest.mark.parametrize("rows,cols", [(1, 32), (1, 896), (15, 96), (16, 128), (17, 160), (33, 4096), (5, 544), (300, 4864)])
def test_quantize(dev, rows, cols):
    """Codes and scale bytes of the 64-bit restatement, and the values back in bf16."""
    from minimal_inference_amd.mxfp4 import quantize_mxfp4

    x = _normals(rows, cols, dev, rows + cols)
    q = quantize_mxfp4(x)
    codes, scales = q.to_codes()
    want_codes, want_scales = omx.quantize(x)
    assert torch.equal(scales.cpu(), want_scales)
    assert torch.equal(codes.cpu(), want_codes)
    assert torch.equal(q.dequantize().double().cpu(), omx.values(want_codes, want_scales))


def test_quantize_every_value(dev):
    """Every bf16 value as the one value of its block and beside a maximum of every
    power of two that rounds it somewhere: ties, saturation, subnormals, zeros,
    infinities and NaN; row strides; the rows around an out are left as they were."""
    from minimal_inference_amd.mxfp4 import quantize_mxfp4

    every = torch.arange(-32768, 32768, device=dev, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    x = torch.zeros(65536, 32, device=dev, dtype=torch.bfloat16)
    x[:, 7] = every
    for j, f in ((0, 1.0), (3, 2.0), (9, -4.0), (31, 1.5)):  # 2 .. 6 times it beside it
        y = x.clone()
        y[:, j] = (every.float() * f).to(torch.bfloat16)
        wide = torch.cat([x, y], 1)
        q = quantize_mxfp4(wide)
        codes, scales = q.to_codes()
        want_codes, want_scales = omx.quantize(wide)
        assert torch.equal(scales.cpu(), want_scales)
        assert torch.equal(codes.cpu(), want_codes)
        out = torch.full((65537, 72), 7.0, device=dev, dtype=torch.bfloat16)
        q.dequantize(out[:-1, :64])
        back, want = out[:-1, :64].double().cpu(), omx.values(want_codes, want_scales)
        assert torch.equal(back.isnan(), want.isnan())
        assert torch.equal(back.nan_to_num(3.0), want.nan_to_num(3.0))
        assert bool((out[-1] == 7).all()) and bool((out[:, 64:] == 7).all())
    strided = torch.cat([x, x], 1)[::3, 32:]
    assert torch.equal(quantize_mxfp4(strided).to_codes()[0], quantize_mxfp4(strided.contiguous()).to_codes()[0])


@pytest.mark.parametrize("rows,cols", [(1, 32), (16, 128), (17, 672), (100, 4096)])
def test_codes_round_trip(dev, rows, cols):
    """from_codes then to_codes returns every byte, scale bytes of 0 and 255 among them."""
    from minimal_inference_amd.mxfp4 import MXFP4

    g = torch.Generator(device=dev).manual_seed(rows * cols)
    codes = torch.randint(0, 256, (rows, cols // 2), device=dev, generator=g, dtype=torch.uint8)
    scales = torch.randint(0, 256, (rows, cols // 32), device=dev, generator=g, dtype=torch.uint8)
    scales[0, 0], scales[-1, -1] = 255, 0
    m = MXFP4.from_codes(codes, scales)
    got = m.to_codes()
    assert torch.equal(got[0], codes) and torch.equal(got[1], scales)


def _bound(x, w, bias, ref):
    """Of one product per entry, before and after its rounding (64 bits)."""
    mag = x.abs() @ w.abs().t() + (0.0 if bias is None else bias.abs())
    return 4 * x.shape[1] ** 0.5 * 2 ** -24 * mag, 2 ** -8 * ref.abs()


ROWS = [1, 3, 15, 16, 17, 32, 33, 64, 65, 127, 128, 129, 200, 300]


@pytest.mark.parametrize("acts", ["bf16", "mxfp4"])
@pytest.mark.parametrize("n,k", [(1, 32), (16, 128), (50, 96), (130, 512), (48, 640), (897, 896), (1152, 4864), (260, 3488)])
@pytest.mark.parametrize("rows", ROWS)
def test_linear(dev, rows, n, k, acts):
    """Odd and ragged sizes on either side of the kernels' tiles, with and without a
    bias, x and out strided; what lies around out's rows stays."""
    from minimal_inference_amd.mxfp4 import linear_mxfp4, quantize_mxfp4

    codes, scales, weight, w = _weight(n, k, dev, n + k)
    g = torch.Generator(device=dev).manual_seed(rows)
    x = torch.randn(rows, k + 64, device=dev, generator=g).to(torch.bfloat16)[:, 32:32 + k]
    if acts == "mxfp4":
        x = quantize_mxfp4(x)
        xd = x.dequantize().double()
    else:
        xd = x.double()
    for bias in (None, torch.randn(n, device=dev, generator=g).to(torch.bfloat16)):
        wide = torch.full((rows + 1, n + 8), 7.0, device=dev, dtype=torch.bfloat16)
        got = linear_mxfp4(x, weight, bias, out=wide[:rows, :n])
        ref = xd @ w.t() + (0.0 if bias is None else bias.double())
        before, after = _bound(xd, w, None if bias is None else bias.double(), ref)
        assert bool(((got.double() - ref).abs() <= before + after).all())
        assert bool((wide[rows] == 7).all()) and bool((wide[:, n:] == 7).all())
        assert torch.equal(linear_mxfp4(x, weight, bias), got)


@pytest.mark.parametrize("acts", ["bf16", "mxfp4"])
@pytest.mark.parametrize("n,k", [(1, 32), (8, 128), (17, 96), (64, 512), (448, 896), (1003, 672)])
@pytest.mark.parametrize("rows", [1, 16, 17, 33, 129, 200])
def test_linear_silu(dev, rows, n, k, acts):
    """The gated product, up rows that begin inside a tile among them.  |silu'| <= 1.1;
    silu and the product in fp32 add 8 roundings of 2^-24."""
    from minimal_inference_amd.mxfp4 import linear_silu_mxfp4, quantize_mxfp4

    codes, scales, weight, w = _weight(2 * n, k, dev, n + k)
    g = torch.Generator(device=dev).manual_seed(rows)
    x = torch.randn(rows, k, device=dev, generator=g).to(torch.bfloat16)
    if acts == "mxfp4":
        x = quantize_mxfp4(x)
    xd = x.double() if acts == "bf16" else x.dequantize().double()
    gate, up = (xd @ w.t()).chunk(2, -1)
    ref = gate * torch.sigmoid(gate) * up
    eg, eu = _bound(xd, w, None, xd @ w.t())[0].chunk(2, -1)
    bound = 1.1 * eg * up.abs() + (gate * torch.sigmoid(gate)).abs() * eu + 1.1 * eg * eu
    wide = torch.full((rows + 1, n + 5), 7.0, device=dev, dtype=torch.bfloat16)
    got = linear_silu_mxfp4(x, weight, out=wide[:rows, :n])
    assert bool(((got.double() - ref).abs() <= bound + (2 ** -8 + 8 * 2 ** -24) * ref.abs()).all())
    assert bool((wide[rows] == 7).all()) and bool((wide[:, n:] == 7).all())
    assert torch.equal(linear_silu_mxfp4(x, weight), got)


@pytest.mark.parametrize("acts", ["bf16", "mxfp4"])
@pytest.mark.parametrize("rows", [1, 16, 32, 64, 150, 260])
@pytest.mark.parametrize("n,k", [(16, 128), (272, 1184), (1040, 2048), (40, 8192), (24, 18944)])
def test_linear_of_whole_numbers(dev, rows, n, k, acts):
    """Whole numbers whose every sum is exact in fp32: the result is the exact one's
    bf16, and a block that is lost or taken twice moves it."""
    from minimal_inference_amd.mxfp4 import linear_mxfp4, quantize_mxfp4

    g = torch.Generator(device=dev).manual_seed(rows + n + k)
    values = torch.tensor([0, 1, 2, 3, 4, 6, -1, -2, -3, -4, -6], device=dev, dtype=torch.float32)

    def whole(r):
        m = values[torch.randint(0, 11, (r, k), device=dev, generator=g)]
        m[:, ::32] = torch.where(m[:, ::32] < 0, -6.0, 6.0)  # every block's scale is 1
        return m.to(torch.bfloat16)

    x, w = whole(rows), whole(n)
    assert 36 * k < 2 ** 24
    weight = quantize_mxfp4(w)
    assert torch.equal(weight.dequantize(), w)
    got = linear_mxfp4(quantize_mxfp4(x) if acts == "mxfp4" else x, weight)
    assert torch.equal(got, (x.double() @ w.double().t()).to(torch.bfloat16))


@pytest.mark.parametrize("acts", ["bf16", "mxfp4"])
@pytest.mark.parametrize("rows", [5, 40])
def test_linear_keeps_infinities_and_nan_in_their_rows(dev, rows, acts):
    """A NaN or an infinity in one row of x or of W reaches that row or column of the
    result alone, also beside k that ends inside a tile; scale byte 255 is NaN."""
    from minimal_inference_amd.mxfp4 import MXFP4, linear_mxfp4, quantize_mxfp4

    n, k = 40, 160
    codes, scales, weight, w = _weight(n, k, dev, 3)
    x = torch.randn(rows, k, device=dev, generator=torch.Generator(device=dev).manual_seed(1)).to(torch.bfloat16)
    x[1, 0], x[3, 159], x[4, 40] = float("inf"), float("nan"), float("-inf")
    make = quantize_mxfp4 if acts == "mxfp4" else (lambda t: t)
    got = linear_mxfp4(make(x), weight).isfinite()
    want = torch.ones(rows, n, dtype=torch.bool, device=dev)
    want[[1, 3, 4]] = False
    # (an infinity times a zero code is NaN and times any other an infinity)
    assert torch.equal(got, want)
    scales[2, 1] = 255
    x = torch.ones(rows, k, device=dev, dtype=torch.bfloat16)
    got = linear_mxfp4(make(x), MXFP4.from_codes(codes, scales)).isnan()
    assert bool(got[:, 2].all()) and int(got.sum()) == rows


def test_linear_far_scales(dev):
    """Scales from 2^-127 up: values at either end of bf16's range times 1, exactly."""
    from minimal_inference_amd.mxfp4 import MXFP4, linear_mxfp4, quantize_mxfp4

    k = 64
    codes = torch.zeros(252, k // 2, dtype=torch.uint8, device=dev)
    codes[:, 0] = 7  # 6 x 2^e in column 0
    scales = torch.arange(252, device=dev, dtype=torch.int32).to(torch.uint8)[:, None].repeat(1, 2)
    w = MXFP4.from_codes(codes, scales)
    want = (6 * torch.exp2(scales[:, 0].double() - 127)).to(torch.bfloat16)
    assert torch.equal(w.dequantize()[:, 0], want)
    x = torch.zeros(2, k, device=dev, dtype=torch.bfloat16)
    x[0, 0] = 1.0
    for rows in (1, 2, 40):
        for xx in (x[:1].repeat(rows, 1), quantize_mxfp4(x[:1].repeat(rows, 1))):
            got = linear_mxfp4(xx, w)
            normal = want.float() >= 2.0 ** -126  # (below, the matrix instructions may flush)
            assert torch.equal(got[0][normal], want[normal])


def test_linear_in_a_graph_and_on_another_stream(dev):
    """Captured and replayed on changed inputs, and called on a side stream: the eager
    results, bit for bit; two calls on two streams at once."""
    from minimal_inference_amd.mxfp4 import linear_mxfp4, linear_silu_mxfp4, quantize_mxfp4

    _, _, w1, _ = _weight(512, 896, dev, 1)
    _, _, w2, _ = _weight(300, 256, dev, 2)
    for rows in (4, 100):
        x = torch.empty(rows, 896, device=dev, dtype=torch.bfloat16)

        def step():
            h = linear_silu_mxfp4(x, w1)
            return h, linear_mxfp4(quantize_mxfp4(h), w2)

        x.normal_()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            first = step()
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(first, step()))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        for seed in range(4):
            x.copy_(torch.randn(rows, 896, generator=torch.Generator().manual_seed(seed)))
            graph.replay()
            held = [t.clone() for t in got]
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(held, step()))
        a, b = torch.cuda.Stream(), torch.cuda.Stream()
        for s in (a, b):
            s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(a):
            ya = [step() for _ in range(8)]
        with torch.cuda.stream(b):
            yb = [step() for _ in range(8)]
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(u, v) for y in ya + yb for u, v in zip(y, want))


def test_one_row_of_any_stride(dev):
    """A single row's stride is not looked at: rows of buffers whose width is odd."""
    from minimal_inference_amd.mxfp4 import linear_mxfp4, quantize_mxfp4

    _, _, w, _ = _weight(33, 64, dev, 8)
    x = torch.randn(1, 64, device=dev).to(torch.bfloat16)
    odd = x.as_strided((1, 64), (3, 1))
    out = torch.empty(33, device=dev, dtype=torch.bfloat16).as_strided((1, 33), (1, 1))
    assert torch.equal(linear_mxfp4(odd, w, out=out), linear_mxfp4(x, w))
    assert torch.equal(quantize_mxfp4(odd).dequantize(), quantize_mxfp4(x).dequantize())


def test_empty_and_refused(dev):
    from minimal_inference_amd.mxfp4 import MXFP4, linear_mxfp4, linear_silu_mxfp4, quantize_mxfp4

    _, _, w, _ = _weight(32, 64, dev, 5)
    x = torch.randn(4, 64, device=dev).to(torch.bfloat16)
    assert linear_mxfp4(x[:0], w).shape == (0, 32)
    assert linear_silu_mxfp4(x[:0], w).shape == (0, 16)
    assert quantize_mxfp4(x[:0]).dequantize().shape == (0, 64)
    assert linear_mxfp4(quantize_mxfp4(x[:0]), w).shape == (0, 32)
    bias = torch.zeros(32, device=dev, dtype=torch.bfloat16)
    odd = torch.zeros(4, 65, device=dev, dtype=torch.bfloat16)[:, 1:]
    far = torch.zeros(1, device=dev, dtype=torch.bfloat16).expand(2, 64)
    square = _weight(64, 64, dev, 7)[2]
    grad = x.clone().requires_grad_()
    for bad in [lambda: linear_mxfp4(x[:, :32], w), lambda: linear_mxfp4(x.float(), w), lambda: linear_mxfp4(odd, w),
                lambda: linear_mxfp4(x, w, bias[:16]), lambda: linear_mxfp4(x, w, bias.float()),
                lambda: linear_mxfp4(x, w, out=x), lambda: linear_mxfp4(x.cpu(), w), lambda: linear_mxfp4(x[0], w),
                lambda: linear_mxfp4(far, w), lambda: linear_mxfp4(x.t().contiguous().t(), w),
                lambda: linear_mxfp4(grad, w), lambda: quantize_mxfp4(grad), lambda: quantize_mxfp4(odd),
                lambda: quantize_mxfp4(x[:, :48]), lambda: quantize_mxfp4(x, out=w), lambda: MXFP4(4, 33, dev),
                lambda: MXFP4.from_codes(torch.zeros(4, 32, dtype=torch.uint8, device=dev),
                                         torch.zeros(4, 1, dtype=torch.uint8, device=dev)),
                lambda: linear_silu_mxfp4(x, _weight(31, 64, dev, 6)[2]), lambda: w.dequantize(x),
                lambda: linear_mxfp4(x, w, bias.clone().requires_grad_()), lambda: linear_mxfp4(x, square, out=x)]:
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        linear_mxfp4(x, x)


@pytest.mark.parametrize("acts", ["bf16", "mxfp4"])
@pytest.mark.parametrize("silu", [False, True])
@pytest.mark.parametrize("rows,n,k", [
    (20, 300, 8192), (33, 520, 2080), (64, 2048, 4096), (65, 130, 18944), (80, 1000, 896), (81, 1000, 4000),
    (128, 640, 8192), (137, 384, 1024), (256, 256, 14336), (265, 4096, 512), (521, 96, 2048), (1024, 2048, 256),
    (2057, 4096, 160), (2304, 3000, 416), (4100, 520, 96), (320, 77, 96), (512, 300, 160), (531, 124, 1184),
    (528, 36, 1184), (649, 80, 6496), (1349, 152, 2624), (2563, 148, 5920), (1432, 34, 3680), (2179, 40, 5440),
    (81, 1773, 7968), (591, 1676, 64), (133, 11615, 64), (165, 10884, 64), (564, 8256, 64), (1205, 6524, 64),
    (528, 7352, 64), (1539, 7712, 64), (1284, 4530, 64), (1290, 916, 7200), (1159, 1028, 7392), (2053, 467, 10080),
    (650, 3891, 3392), (2563, 3116, 672), (1295, 6303, 544), (4671, 1788, 1216), (4124, 4007, 928),
    (263, 1836, 64), (288, 5555, 64), (1281, 5936, 64), (771, 4957, 64), (1923, 2064, 544), (2568, 1588, 704),
    (4109, 916, 1216), (1671, 1179, 1664), (1284, 2040, 3520), (645, 1878, 4032), (1295, 1004, 6560),
    (646, 1020, 8224), (1538, 385, 7424), (2621, 3078, 1056), (3360, 4820, 1088), (4127, 2019, 2080),
    (4657, 858, 2144), (3596, 1060, 4064), (3604, 554, 3584), (648, 1936, 7808), (2307, 1688, 2752), (24, 76, 13120),
    (79, 50, 4128), (92, 84, 11616)])
def test_every_form_of_whole_numbers(dev, rows, n, k, silu, acts):
    """Sizes on which the forms (groups of 32 or 64 rows, blocks of 32 to 256 rows, k
    whole and in parts, rows behind the last whole block) differ: sums exact in fp32 are the exact ones, with a
    workspace and without one, strided rows and what lies around them included."""
    from minimal_inference_amd import _lib
    from minimal_inference_amd.mxfp4 import linear_mxfp4, linear_silu_mxfp4, quantize_mxfp4

    g = torch.Generator(device=dev).manual_seed(rows + n + k)
    values = torch.tensor([0, 1, 2, 3, 4, 6, -1, -2, -3, -4, -6], device=dev, dtype=torch.float32)

    def whole(r):
        m = values[torch.randint(0, 11, (r, k), device=dev, generator=g)]
        m[:, ::32] = torch.where(m[:, ::32] < 0, -6.0, 6.0)
        return m.to(torch.bfloat16)

    x, w = whole(rows), whole(2 * n if silu else n)
    weight = quantize_mxfp4(w)
    xx = quantize_mxfp4(x) if acts == "mxfp4" else torch.cat([x, torch.full_like(x[:, :32], float("nan"))], 1)[:, :k]
    sums = x.double() @ w.double().t()
    ref = sums
    if silu:
        gate, up = sums.chunk(2, -1)
        ref = gate * torch.sigmoid(gate) * up
    out = torch.full((rows + 1, n + 8), 7.0, device=dev, dtype=torch.bfloat16)
    (linear_silu_mxfp4 if silu else linear_mxfp4)(xx, weight, out=out[:rows, :n])
    alone = torch.full_like(out, 7.0)  # and by the C entry, which may get no workspace
    ptr = (xx.codes_ptr, 0, xx.scales_ptr) if acts == "mxfp4" else (xx.data_ptr(), xx.stride(0), None)
    _lib.call("mi_linear_mxfp4", *ptr, weight.codes_ptr, weight.scales_ptr, None, alone.data_ptr(), alone.stride(0), rows, n,
              k, int(silu), None, 0, torch.cuda.current_stream().cuda_stream)
    for got in (out, alone):
        if silu:  # fp32: the exponential, the quotient and the products round 8 times
            assert bool(((got[:rows, :n].double() - ref).abs() <= (2 ** -8 + 8 * 2 ** -24) * ref.abs() + 1e-30).all())
        else:
            assert torch.equal(got[:rows, :n], ref.to(torch.bfloat16))
        assert bool((got[rows] == 7).all()) and bool((got[:, n:] == 7).all())


@pytest.mark.parametrize("silu", [False, True])
@pytest.mark.parametrize("rows,acts", [(1, "bf16"), (20, "bf16"), (7, "mxfp4"), (20, "mxfp4"), (40, "mxfp4"), (64, "mxfp4")])
@pytest.mark.parametrize("k", [160, 3616])
@pytest.mark.parametrize("w_rows", [4000, 8190, 10_234, 16_002, 18_420, 22_004, 28_660, 32_002, 40_006, 59_000, 70_002])
def test_few_rows_of_every_width(dev, w_rows, k, rows, acts, silu):
    """One to eight tiles of W per workgroup, one round of them and several, four waves
    and eight: whole numbers whose sums are exact in fp32."""
    from minimal_inference_amd.mxfp4 import MXFP4, linear_mxfp4, linear_silu_mxfp4, quantize_mxfp4

    g = torch.Generator(device=dev).manual_seed(rows + w_rows + k)
    values = torch.tensor([0, 1, 2, 3, 4, 6, -1, -2, -3, -4, -6], device=dev, dtype=torch.bfloat16)
    x = values[torch.randint(0, 11, (rows, k), device=dev, generator=g)]
    x[:, ::32] = 6.0
    codes = torch.randint(0, 256, (w_rows, k // 2), device=dev, generator=g, dtype=torch.uint8)
    weight = MXFP4.from_codes(codes, torch.full((w_rows, k // 32), 128, device=dev, dtype=torch.uint8))
    sums = x.float() @ weight.dequantize().float().t()  # (whole numbers below 2^24)
    xx = quantize_mxfp4(x) if acts == "mxfp4" else x
    if silu:
        gate, up = sums.double().chunk(2, -1)
        ref = gate * torch.sigmoid(gate) * up
        got = linear_silu_mxfp4(xx, weight).double()  # fp32: 8 roundings, then one to bf16
        assert bool(((got - ref).abs() <= (2 ** -8 + 8 * 2 ** -24) * ref.abs() + 1e-30).all())
    else:
        assert torch.equal(linear_mxfp4(xx, weight), sums.to(torch.bfloat16))
