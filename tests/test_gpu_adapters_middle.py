"""GPU: A x enters the second product as 16 bits, held with y's rounding out of the way.

y is -bf16(scale B A x), so that what is rounded to bf16 at the end is that number's own rounding, 2^-9 of it: the bar
(that of test_gpu_adapters) is then 2^-16 of A x and fp32 sums, and a product with A x in bf16 alone does not pass.
"""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_adapters import _make, _want

pytestmark = pytest.mark.gpu


# one launch; few rows by shared units and by a wave's own; tiles of 64 rows; ranks of every size of launch
@pytest.mark.parametrize("x8", [False, True])
@pytest.mark.parametrize("rows,slots,k,pieces,rank", [(3, 2, 896, [304], 16), (40, 20, 4096, [96, 32], 8), (17, 3, 8192, [304], 16), (300, 40, 544, [4864], 32),
                                                      (64, 5, 1056, [160, 160], 64), (400, 3, 4864, [896, 128], 16), (700, 9, 1056, [304], 64),
                                                      (333, 2, 256, [160, 96], 128)])
def test_sixteen_bits_of_the_middle(dev, rows, slots, k, pieces, rank, x8):
    from minimal_inference_amd.adapters import AdapterPlan, add_adapters

    x, values, ad, slot, y = _make(dev, rows, k, pieces, rank, slots, x8=x8)
    zero = torch.zeros_like(y)
    y = (-_want(values, ad, slot, zero)[0]).float().to(torch.bfloat16)
    ref, tol = _want(values, ad, slot, y)
    plan = AdapterPlan(rows, slots, dev)
    plan.plan(slot)
    got = add_adapters(y, x, ad, plan, out=torch.empty_like(y)).double()
    assert bool(((got - ref).abs() <= tol).all())
    # (eight bits of A x would not pass: some entry is further off; along a long k the bar is mostly fp32's)
    coarse = y.double().clone()
    for s in range(slots):
        mine, first = (slot == s).nonzero()[:, 0], 0
        v = ((values[mine] @ ad.a[s].double().t()) * ad.scale[s].double()).float().to(torch.bfloat16).double()
        for i, n in enumerate(pieces):
            coarse[mine, first: first + n] += v[:, i * rank: (i + 1) * rank] @ ad.b[s, first: first + n].double().t()
            first += n
    assert bool(((coarse - ref).abs() > tol).any())
