"""GPU: the filtered draw at the ends of its ranges: uniform numbers of zero and next to
it, over every form of its launches, against the same draw in 64 bits.

Ids are equal.  Both sides sum the kept weights in index order in 64 bits and compare with
u times the total; each sum of n positive terms is within n 2^-53 of the exact one
relative to itself, so a draw differs only where u times the total lies within some
2^-33 (n = 2^20), relative to itself, of a border.
"""

from __future__ import annotations

import math

import pytest
import torch

from oracle.draw import draw_row

pytestmark = pytest.mark.gpu


def _uniform(n, dev, seed):
    return torch.rand(n, device=dev, generator=torch.Generator(device=dev).manual_seed(seed))


def _logits(b, v, dev, seed, spread=3.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(b, v, device=dev, generator=g) * spread).to(torch.bfloat16)


def _check(dev, logits, u, temperature, top_p=None, top_k=None, min_p=None):
    from minimal_inference_amd.sampling import Sampler

    b, v = logits.shape
    s = Sampler(dev, b, vocab=v)
    s.set_params(temperature, top_p, top_k=top_k, min_p=min_p)
    got = s.draw(logits, u).tolist()
    host, uh = logits.cpu(), u.cpu().double().tolist()
    f32 = lambda x: torch.tensor(x, dtype=torch.float32).double().tolist()  # noqa: E731
    t, p, m = f32(temperature), f32(top_p or [1.0] * b), f32(min_p or [0.0] * b)
    k = top_k or [0] * b
    assert got == [draw_row(host[i], uh[i], t[i], k[i], p[i], m[i]) for i in range(b)]


@pytest.mark.parametrize("v", [100, 5000, 20000, 40000, 152064])
def test_zero_and_small_u_beside_low_values(dev, v):
    """Values from -2^8 down that weigh next to nothing, at the row's begin: at u = 0 the
    first of them is drawn as long as its weight is above zero in 64 bits, at small u one
    of those that reach it, else the row's middle."""
    b = 16
    logits = torch.full((b, v), -300.0, device=dev, dtype=torch.bfloat16)
    logits[:, v // 2] = 0.0
    logits[8:12, : v // 2] = -1000.0
    logits[12:14, : v // 4] = torch.finfo(torch.bfloat16).min  # (weighs nothing at any of these temperatures)
    logits[14:, ::3] = -256.0
    t = [5.0, 5.0, 3.0, 3.0, 2.0, 1.0, 0.5, 0.3] * 2
    for u in (0.0, 1e-35, 1e-30, 2.0 ** -60, 2.0 ** -44, 2.0 ** -24, 0.3):
        uniforms = torch.full((b,), u, device=dev)
        _check(dev, logits, uniforms, t)
        _check(dev, logits, uniforms, t, top_k=[0, 1, 2, v // 2] * 4, top_p=[1.0, 1.0, 0.9, 1.0] * 4,
               min_p=[0.0, 0.0, 0.0, 1e-30] * 4)


@pytest.mark.parametrize("v", [100, 40000])
def test_small_u_inside_a_lane(dev, v):
    """u between the sums of tokens that weigh next to nothing, some of them beside one
    that holds nearly all of the weight."""
    logits = torch.full((64, v), -200.0, device=dev, dtype=torch.bfloat16)
    u = torch.empty(64, dtype=torch.float64)
    for i in range(64):
        logits[i, : i + 1] = -80.0
        logits[i, i + 1] = 0.0
        u[i] = (i + 0.5) * math.exp(-80.0)  # the last of those i + 1
    _check(dev, logits, u.float().to(dev), [1.0] * 64)
    _check(dev, logits, (u / 2).float().to(dev), [1.0] * 64, min_p=[1e-35] * 64)
    _check(dev, logits, u.float().to(dev), [1.0] * 64, top_k=[50] * 64)


@pytest.mark.parametrize("b,v", [(3, 500), (2, 50000)])
def test_first_draw_of_a_sampler_in_a_graph(dev, b, v):
    """A sampler that knows its vocabulary is ready for a captured draw as it stands."""
    from minimal_inference_amd.sampling import Sampler

    s = Sampler(dev, b, vocab=v)
    s.set_params([0.9] * b, [0.9] * b, top_k=[40] * b, min_p=[0.01] * b)
    logits, u = _logits(b, v, dev, 1), _uniform(b, dev, 2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ids = s.draw(logits, u)
    f = lambda x: torch.tensor(x).double().item()  # noqa: E731
    for seed in range(3):
        logits.copy_(_logits(b, v, dev, 10 + seed))
        u.copy_(_uniform(b, dev, 20 + seed))
        graph.replay()
        held = ids.tolist()
        assert held == [draw_row(logits[i].cpu(), u[i].item(), f(0.9), 40, f(0.9), f(0.01)) for i in range(b)]
        assert s.draw(logits, u).tolist() == held
