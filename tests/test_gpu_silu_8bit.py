"""GPU: silu of the 8-bit gated product, held against the 2^-20 that its kernels state.

Each output is brought to just beside the middle between two e4m3 codes, on either side of it: 2^-20 (silu) and 2^-23 (the
product's own rounding, 2^-24, and as much again), relative.  Its code then says on which side the kernel's fp32 value lies.
Gates and ups are any fp32 numbers: six pieces of four bits, a code each under a power of two of its own, whose
sum is exact.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

K = 256  # eight blocks, six of them used


def _pieces(v):
    """Codes (whole numbers up to 15) and scale bytes whose sum is the fp32 number v, |v| from 2^-100 up."""
    m, e = np.frexp(np.float64(v))
    whole = int(abs(m) * 2 ** 24)
    assert whole == abs(m) * 2 ** 24
    codes, scales = np.zeros(8), np.full(8, 127)
    for i in range(6):
        codes[i] = (whole >> (20 - 4 * i) & 15) * np.sign(m)
        scales[i] = 127 + e - 24 + 20 - 4 * i
    assert scales.min() >= 0 and scales.max() <= 254
    return codes, scales


def _silu(g):
    g = np.longdouble(g)
    return g / (1 + np.exp(-g))


# (the codes of a block are of 2^9 to 2^16 times the unit's 1: its largest sets the unit)
@pytest.mark.parametrize("gates", [(-0.013, -0.5, -1.0, -3.3), (-7.7, -15.1, -30.0, -42.42), (-50.0, -55.5, -60.1, -64.3), (-70.0, -77.7, -80.0, -86.0),
                                   (0.013, 0.7, 2.2, 9.9), (17.3, 33.0, 64.1, 86.0)])
def test_silu_within_its_bound(dev, gates):
    from minimal_inference_amd.mxfp8 import MXFP8, linear_silu_mxfp8

    rng = np.random.default_rng(7)
    delta = 2.0 ** -20 + 2.0 ** -23
    gate, up, want = [], [], []
    for base in gates:
        for j in range(8):  # blocks of a gate and its neighbours
            g = np.float32(base * (1 + 0.01 * rng.random()))
            silu = _silu(g)
            gate += [g] * 32
            up.append(np.float32(400 / silu))  # sets the unit to 1
            want.append(None)
            for _ in range(31):
                step = 2.0 ** rng.integers(-2, 6)  # of codes 8 step .. 16 step
                low = step * rng.integers(8, 16)  # (up to 480 of 448: the largest code takes no part)
                if low + step > 416:
                    low = 8.0 * step
                middle, side = np.longdouble(low + step / 2), rng.choice([-1, 1])
                u = np.float32(middle / silu * (1 + side * np.longdouble(delta)))
                exact = silu * np.longdouble(u)
                if abs(exact / middle - 1) < np.longdouble(delta) - np.longdouble(2) ** -25:  # (u's rounding: one step further)
                    u = np.nextafter(u, np.float32(np.inf) if side * np.sign(u) > 0 else np.float32(-np.inf), dtype=np.float32)
                    exact = silu * np.longdouble(u)
                assert (exact / middle - 1) * side >= np.longdouble(2) ** -20 + np.longdouble(2) ** -24
                up.append(u)
                want.append(low + step if side > 0 else low)
    n = len(gate)
    codes, scales = np.zeros((2 * n, K), np.float32), np.zeros((2 * n, 8), np.uint8)
    for row, v in enumerate(gate + up):
        codes[row, ::32], scales[row] = _pieces(v)
    weight = MXFP8.from_codes(torch.tensor(codes).to(torch.float8_e4m3fn).to(dev), torch.tensor(scales).to(dev))
    x = torch.zeros(1, K)
    x[0, ::32] = 1.0
    for rows in (1, 200, 300):  # (few rows, blocks, the largest blocks)
        m = MXFP8.from_codes(x.expand(rows, K).to(torch.float8_e4m3fn).contiguous().to(dev),
                             torch.full((rows, 8), 127, dtype=torch.uint8, device=dev))
        q = linear_silu_mxfp8(m, weight, quantize=True)
        assert bool((q.scales == 127).all())
        got = q.codes.float().cpu().numpy()
        wrong = [(gate[i], want[i], float(got[0, i])) for i in range(n) if want[i] is not None and got[0, i] != want[i]]
        assert not wrong, (rows, len(wrong), wrong[:4])
        assert (got == got[:1]).all()
