"""GPU: codes of the 8-bit norm where x w / rms lies within 3e-8 of the middle of two codes and the product of x w with
the rounded root lies on its other side."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import mxfp8 as om8

pytestmark = pytest.mark.gpu

EPS = 1e-6
# (seed of the row's other elements, mantissas of x and w in 128ths), found by search on the CPU
CASES = [(638, 162, 164), (638, 164, 174), (638, 164, 186), (638, 216, 246), (638, 232, 246), (638, 246, 248), (3202, 220, 241),
         (5483, 239, 255), (11839, 218, 226), (28898, 142, 173), (31982, 231, 247), (33445, 235, 243)]


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("seed,a,b", CASES)
def test_codes_beside_a_middle(dev, seed, a, b, sign):
    from minimal_inference_amd.mxfp8 import add_rms_norm_mxfp8

    x = np.concatenate([np.arange(128, 256) / 128, np.random.default_rng(seed).integers(96, 144, 256) / 256])
    root = 1 / np.sqrt(np.square(x).mean() + np.float64(np.float32(EPS)))
    exact, near = a * b / 2 ** 14 * root, float(np.float32(a * b / 2 ** 14) * np.float32(root))
    half = 2.0 ** (np.floor(np.log2(exact)) - 4)
    middle = np.rint(exact / half) * half
    assert np.rint(exact / half) % 2 == 1 and (exact > middle) != (near > middle)  # (such a case indeed)
    x = torch.tensor(x * sign)
    w = torch.full((384,), b / 128, dtype=torch.bfloat16)
    want = om8.quantize((x * (b / 128) * root)[None])
    xs = x.to(torch.bfloat16)
    assert torch.equal(xs.double(), x)
    q = add_rms_norm_mxfp8(xs[None].to(dev), None, w.to(dev), EPS)
    assert torch.equal(q.scales.cpu(), want[1])
    assert torch.equal(q.codes.view(torch.uint8).cpu(), want[0])
