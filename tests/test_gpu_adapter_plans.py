"""GPU: plans that follow each other in one buffer."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [5, 400])
def test_replay_after_a_plan_of_no_rows(dev, rows):
    """A captured call finds another number of rows than its own, none, and leaves NaN; its own plan brings its
    own bits back."""
    from minimal_inference_amd.adapters import AdapterPlan, Adapters, add_adapters

    g = torch.Generator(device=dev).manual_seed(rows)
    rand = lambda *s: torch.randn(*s, device=dev, generator=g).to(torch.bfloat16)  # noqa: E731
    ad = Adapters(rand(2, 8, 64), rand(2, 48, 8), torch.ones(2, device=dev), [48])
    x, y = rand(rows, 64), rand(rows, 48)
    slot = (torch.arange(rows, device=dev) % 3 - 1).to(torch.int32)
    plan = AdapterPlan(rows, 2, dev)
    plan.plan(slot)
    want, got = add_adapters(y, x, ad, plan, out=torch.empty_like(y)), torch.empty_like(y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        add_adapters(y, x, ad, plan, out=got)
    for _ in range(3):
        plan.plan(slot[:0])
        assert plan.rows == 0
        graph.replay()
        assert bool(got.isnan().all())
        plan.plan(slot)
        graph.replay()
        assert torch.equal(got, want)
