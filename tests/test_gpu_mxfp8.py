"""GPU: MXFP8 matrices, the norm that leaves them and the linear layers over them against
64-bit restatements.

Bars.  Quantisation and the return to bf16 are exact.  Of a product: the matrix instruction
cuts products at 2^-13 of the largest that it adds with them, some 16 at a time; independent errors of
up to that stay within 2^-10 of the 2-norm of the entry's products (7 standard deviations), and the
sum is rounded once to bf16 (2^-8 relative).  Whole numbers of few bits are summed
exactly.  The norm's codes are those of the exact norm: its error before the one rounding is that of 64
bits (and of a pair of fp32 numbers for the root, 2^-48), which meets a border with a chance of 1e-13 a value.
"""

from __future__ import annotations

import pytest
import torch

from oracle import mxfp8 as om8

pytestmark = pytest.mark.gpu


def _normals(rows, cols, dev, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn(rows, cols, device=dev, generator=g)
    return (x * torch.exp(2 * torch.randn(rows, 1, device=dev, generator=g))).to(torch.bfloat16)


def _matrix(n, k, dev, seed):
    """A random MXFP8 matrix and its values in 64 bits."""
    from minimal_inference_amd.mxfp8 import MXFP8

    g = torch.Generator(device=dev).manual_seed(seed)
    v = torch.randn(n, k, device=dev, generator=g).mul_(100).clamp_(-448, 448)
    codes = v.to(torch.float8_e4m3fn)
    scales = torch.randint(118, 124, (n, k // 32), device=dev, generator=g, dtype=torch.uint8)
    return MXFP8.from_codes(codes, scales), om8.values(codes, scales)


@pytest.mark.parametrize("rows,cols", [(1, 32), (1, 896), (15, 96), (16, 128), (17, 160), (33, 4096), (5, 544), (300, 4864)])
def test_quantize(dev, rows, cols):
    """Codes and scale bytes of the 64-bit restatement, and the values back in bf16."""
    from minimal_inference_amd.mxfp8 import quantize_mxfp8

    x = _normals(rows, cols, dev, rows + cols)
    q = quantize_mxfp8(x)
    codes, scales = om8.quantize(x)
    assert torch.equal(q.scales.cpu(), scales)
    assert torch.equal(q.codes.view(torch.uint8).cpu(), codes)
    assert torch.equal(q.dequantize().double().cpu(), om8.values(codes, scales))


def test_quantize_every_value(dev):
    """Every bf16 value as the one value of its block and beside a maximum of other powers of two and
    mantissas: ties, borders of the power, subnormals, zeros, infinities and NaN; row strides; what
    lies around an out is left as it was."""
    from minimal_inference_amd.mxfp8 import MXFP8, quantize_mxfp8

    every = torch.arange(-32768, 32768, device=dev, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    x = torch.zeros(65536, 32, device=dev, dtype=torch.bfloat16)
    x[:, 7] = every
    for j, f in ((0, 1.0), (3, 1.75), (9, -1.765625), (31, 300.0), (30, 2.0 ** 14)):
        y = x.clone()
        y[:, j] = (every.float() * f).to(torch.bfloat16)
        wide = torch.cat([x, y], 1)
        q = quantize_mxfp8(wide)
        codes, scales = om8.quantize(wide)
        assert torch.equal(q.scales.cpu(), scales)
        assert torch.equal(q.codes.view(torch.uint8).cpu(), codes)
        out = torch.full((65537, 72), 7.0, device=dev, dtype=torch.bfloat16)
        q.dequantize(out[:-1, :64])
        want = om8.values(codes, scales)
        back = out[:-1, :64].cpu()
        # the least values are below bf16's least: its nearest then
        assert torch.equal(back.double().nan_to_num(3.0), want.float().to(torch.bfloat16).double().nan_to_num(3.0))
        assert torch.equal(back.isnan(), want.isnan())
        assert bool((out[-1] == 7).all()) and bool((out[:, 64:] == 7).all())
    strided = torch.cat([x, x], 1)[::3, 32:]
    assert torch.equal(quantize_mxfp8(strided).codes.view(torch.uint8), quantize_mxfp8(strided.contiguous()).codes.view(torch.uint8))
    room = torch.full((65536, 64 + 48), 9, device=dev, dtype=torch.uint8)
    held = MXFP8.from_codes(room[:, :64], torch.zeros(65536, 16, device=dev, dtype=torch.uint8)[:, :2])
    quantize_mxfp8(wide, held)
    assert torch.equal(held.codes.view(torch.uint8).cpu(), codes)


def test_every_code_back(dev):
    """Every code under every scale byte."""
    from minimal_inference_amd.mxfp8 import MXFP8

    codes = torch.arange(256, device=dev, dtype=torch.uint8).repeat(256, 1)
    scales = torch.arange(256, device=dev, dtype=torch.uint8)[:, None].repeat(1, 8)
    back = MXFP8.from_codes(codes, scales).dequantize()
    want = om8.values(codes, scales).float().to(torch.bfloat16)
    assert torch.equal(back.isnan(), want.isnan())
    assert torch.equal(back.nan_to_num(3.0), want.nan_to_num(3.0))


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("rows,hidden", [(1, 32), (1, 896), (3, 4096), (48, 8192), (17, 96), (5, 16384), (130, 544), (2, 12320)])
def test_add_rms_norm(dev, rows, hidden, delta):
    """The sum's bits; the codes and scales of the exact norm; the same in place, into an out, over strided
    rows."""
    from minimal_inference_amd.mxfp8 import MXFP8, add_rms_norm_mxfp8

    g = torch.Generator(device=dev).manual_seed(rows * hidden)
    x = _normals(rows, hidden, dev, hidden)
    d = torch.randn(rows, hidden, device=dev, generator=g).to(torch.bfloat16) if delta else None
    w = (1 + 0.1 * torch.randn(hidden, device=dev, generator=g)).to(torch.bfloat16)
    s = x if d is None else x + d
    v = s.double()
    h = v / (v.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
    x_out = torch.empty_like(x)
    q = add_rms_norm_mxfp8(x, d, w, 1e-6, x_out=x_out)
    assert torch.equal(x_out, s)
    codes, scales = om8.quantize(h)
    assert torch.equal(q.scales.cpu(), scales)
    assert torch.equal(q.codes.view(torch.uint8).cpu(), codes)
    # the same elsewhere: into an out whose rows are strided, from strided rows, in place
    wide = torch.zeros(rows, 3 * hidden, device=dev, dtype=torch.bfloat16)
    wide[:, hidden: 2 * hidden] = x
    out = MXFP8(rows, hidden, dev)
    x2 = wide[:, hidden: 2 * hidden]
    assert add_rms_norm_mxfp8(x2, d, w, 1e-6, out=out) is out
    assert torch.equal(x2, s) and not bool(wide[:, :hidden].any()) and not bool(wide[:, 2 * hidden:].any())
    assert torch.equal(out.codes.view(torch.uint8), q.codes.view(torch.uint8)) and torch.equal(out.scales, q.scales)


def test_add_rms_norm_of_extremes(dev):
    """Rows of zeros, of the largest and the least values and with an infinity or a NaN: blocks that are NaN as a
    whole; squares that leave fp32's range."""
    from minimal_inference_amd.mxfp8 import add_rms_norm_mxfp8

    x = torch.ones(6, 128, device=dev, dtype=torch.bfloat16)
    x[0] = 0
    x[1] = 3e38
    x[4] = 1e-38
    x[5, ::2], x[5, 1::2] = 1e-30, 1e30
    x[2, 40] = float("inf")
    x[3, 100] = float("nan")
    w = torch.ones(128, device=dev, dtype=torch.bfloat16)
    q = add_rms_norm_mxfp8(x, None, w, 1e-6)
    v = q.dequantize()
    assert bool((v[0] == 0).all())
    rows = [1, 4, 5]
    d = x[rows].double()
    codes, scales = om8.quantize(d / (d.square().mean(-1, keepdim=True) + 1e-6).sqrt())
    assert torch.equal(q.codes.view(torch.uint8)[rows].cpu(), codes) and torch.equal(q.scales[rows].cpu(), scales)
    tiny = add_rms_norm_mxfp8(x[4:5], None, w, 0.0).dequantize()
    assert bool((tiny == 1).all())
    assert bool(v[2, 32:64].isnan().all()) and bool((v[2, :32] == 0).all()) and bool(v[3].isnan().all())


def _bound(x, w, ref):
    """Of one product per entry, before and after its rounding (64 bits)."""
    return 2.0 ** -10 * (x.square() @ w.square().t()).sqrt(), 2 ** -8 * ref.abs()


ROWS = [1, 3, 15, 16, 17, 32, 33, 64, 65, 127, 128, 129, 200, 300]


@pytest.mark.parametrize("n,k", [(1, 32), (16, 128), (50, 96), (130, 512), (48, 640), (897, 896), (1152, 4864), (260, 3488)])
@pytest.mark.parametrize("rows", ROWS)
def test_linear(dev, rows, n, k):
    """Odd and ragged sizes on either side of the kernels' tiles, with and without a bias; what
    lies around out's rows stays."""
    from minimal_inference_amd.mxfp8 import linear_mxfp8

    weight, w = _matrix(n, k, dev, n + k)
    m, x = _matrix(rows, k, dev, rows)
    for bias in (None, torch.randn(n, device=dev, generator=torch.Generator(device=dev).manual_seed(k)).to(torch.bfloat16)):
        ref = x @ w.t()
        pre, _ = _bound(x, w, ref)
        if bias is not None:
            ref = ref + bias.double()
        tol = pre + 2 ** -8 * (ref.abs() + pre)
        got = linear_mxfp8(m, weight, bias)
        assert bool(((got.double() - ref).abs() <= tol).all())
        room = torch.full((rows, n + 13), 7.0, device=dev, dtype=torch.bfloat16)
        assert linear_mxfp8(m, weight, bias, room[:, 5: 5 + n]) .data_ptr() == room[:, 5:].data_ptr()
        assert torch.equal(room[:, 5: 5 + n], got)
        assert bool((room[:, :5] == 7).all()) and bool((room[:, 5 + n:] == 7).all())


@pytest.mark.parametrize("rows", [1, 40, 64, 100, 128, 300, 777])
@pytest.mark.parametrize("n,k", [(32, 32), (96, 224), (544, 1056), (128, 8192)])
def test_linear_of_whole_numbers(dev, rows, n, k):
    """Whole numbers up to 8 with powers of two within 2^3: every sum is exact in fp32, so out is the
    exact sum's rounding, bit for bit, wherever k is cut."""
    from minimal_inference_amd.mxfp8 import MXFP8, linear_mxfp8

    g = torch.Generator(device=dev).manual_seed(rows + n)

    def whole(r):
        codes = torch.randint(-8, 9, (r, k), device=dev, generator=g).float().to(torch.float8_e4m3fn)
        scales = torch.randint(126, 129, (r, k // 32), device=dev, generator=g, dtype=torch.uint8)
        return MXFP8.from_codes(codes, scales), om8.values(codes, scales)

    (m, x), (weight, w) = whole(rows), whole(n)
    assert torch.equal(linear_mxfp8(m, weight), (x @ w.t()).float().to(torch.bfloat16))


@pytest.mark.parametrize("rows", [1, 17, 64, 65, 128, 200, 300])
@pytest.mark.parametrize("n,k", [(16, 32), (32, 128), (50, 96), (160, 640), (864, 896), (1056, 3488)])
def test_linear_silu(dev, rows, n, k):
    """The gated product in bf16, and, in blocks of 32, in 8 bits: codes that are those of some value as
    near to the exact one as the sums are."""
    from minimal_inference_amd.mxfp8 import linear_silu_mxfp8

    weight, w = _matrix(2 * n, k, dev, n + k)
    m, x = _matrix(rows, k, dev, rows)
    w = w * 2.0 ** -6  # (gates of a few units)
    weight.scales.copy_(weight.scales - 6)
    gate, up = (x @ w.t()).chunk(2, -1)
    eg, eu = _bound(x, w, gate)[0].chunk(2, -1)
    ref = gate * torch.sigmoid(gate) * up
    # silu's slope is at most 1.1
    pre = 1.1 * eg * (up.abs() + eu) + (gate * torch.sigmoid(gate)).abs() * eu + 2.0 ** -21 * ref.abs()
    got = linear_silu_mxfp8(m, weight)
    assert bool(((got.double() - ref).abs() <= pre + 2 ** -8 * (ref.abs() + pre)).all())
    if n % 32:
        return
    q = linear_silu_mxfp8(m, weight, quantize=True)
    v = om8.values(q.codes, q.scales)
    unit = torch.exp2(q.scales.double() - 127).repeat_interleave(32, 1)
    # half a step of e4m3: 2^-4 of the value, 2^-10 of the unit below 2^-6 of it
    assert bool(((v - ref).abs() <= pre + torch.maximum(2 ** -4 * (ref.abs() + pre), 2 ** -10 * unit)).all())
    amax = (ref.abs() + pre).view(rows, n // 32, 32).amax(-1)
    least = (ref.abs() - pre).view(rows, n // 32, 32).amax(-1)
    u = unit[:, ::32]
    assert bool((448 * u >= least).all()) and bool(((224 * u <= amax) | (q.scales == 0)).all())


def test_scales_padding_is_not_read_into_the_sum(dev):
    """Scale rows whose bytes behind the last block are NaN's, codes behind k that are NaN."""
    from minimal_inference_amd.mxfp8 import MXFP8, linear_mxfp8

    for rows in (5, 100, 300):
        m, x = _matrix(rows, 160, dev, rows)
        weight, w = _matrix(96, 160, dev, 1)
        want = linear_mxfp8(m, weight)
        wide = torch.full((rows, 256), 127, device=dev, dtype=torch.uint8)  # NaN
        wide[:, :160] = m.codes.view(torch.uint8)
        scales = torch.full((rows, 16), 255, device=dev, dtype=torch.uint8)
        scales[:, :5] = m.scales
        other = MXFP8(rows, 160, dev)
        other.anchor.fill_(255)
        other.codes.view(torch.uint8).copy_(wide[:, :160])
        other.scales.copy_(scales[:, :5])
        held = MXFP8(rows, 160, dev)
        held.anchor, held.codes_ptr, held.codes_stride = wide, wide.data_ptr(), 256
        held.scales_ptr, held.scales_stride = scales.data_ptr(), 16
        for y in (other, held):
            assert torch.equal(linear_mxfp8(y, weight), want)


def test_infinities_and_nan_stay_in_their_rows(dev):
    from minimal_inference_amd.mxfp8 import linear_mxfp8

    for rows in (7, 100, 400):
        m, _ = _matrix(rows, 256, dev, rows)
        weight, _ = _matrix(64, 256, dev, 2)
        want = linear_mxfp8(m, weight)
        m.scales[3, 5] = 255
        m.codes.view(torch.uint8)[5, 200] = 127
        got = linear_mxfp8(m, weight)
        rest = [i for i in range(rows) if i not in (3, 5)]
        assert bool(got[3].isnan().all()) and bool(got[5].isnan().all())
        assert torch.equal(got[rest], want[rest])


def test_from_codes_holds_or_copies(dev):
    from minimal_inference_amd.mxfp8 import MXFP8

    codes = torch.randint(0, 120, (9, 1024), device=dev, dtype=torch.uint8)
    scales = torch.randint(100, 140, (9, 32), device=dev, dtype=torch.uint8)
    m = MXFP8.from_codes(codes, scales)
    assert m.codes_ptr == codes.data_ptr() and m.scales_ptr == scales.data_ptr()
    for c, s in ((codes[:, :96], scales[:, :3]), (codes[:, 1:97], scales[:, 1:4]), (codes[::2, 32:], scales[::2, 1:]),
                 (codes.view(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu))):
        m = MXFP8.from_codes(c, s)
        assert torch.equal(m.codes.view(torch.uint8), c.view(torch.uint8)) and torch.equal(m.scales, s.view(torch.uint8))
        assert torch.equal(m.dequantize().double(), om8.values(c.contiguous(), s.contiguous()))
