"""CPU: what the operators over 4-bit matrices and around blocks refuse before a launch."""

from __future__ import annotations

import pytest
import torch


def test_derivatives():
    from torch.autograd import forward_ad

    from minimal_inference_amd._util import refuse_derivatives

    x = torch.randn(4)
    refuse_derivatives("x", None)
    refuse_derivatives("x", x)
    with pytest.raises(ValueError, match="gradient"):
        refuse_derivatives("x", x.clone().requires_grad_())
    with torch.no_grad():
        refuse_derivatives("x", x.clone().requires_grad_())
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones(4))
        for t in (dual, dual[1:], dual * 2):
            with pytest.raises(ValueError, match="tangent"):
                refuse_derivatives("x", t)
        refuse_derivatives("x", x)
        with torch.inference_mode():
            refuse_derivatives("x", dual)
    refuse_derivatives("x", dual)
