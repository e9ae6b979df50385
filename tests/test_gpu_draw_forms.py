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


# (rows, vocabulary) of two launches: workgroups of 8,192 tokens up to 8 of them, of 16,384 up to
# 32, and of 32,768 from 256 workgroups of the others on and up to 32, the last of them whole or not
TWO_LAUNCHES = [(2, 65536), (3, 65530), (3, 200000), (2, 524288), (24, 180225), (48, 152064), (48, 151929), (30, 151929),
                (64, 65536), (20, 400003), (2, 524289), (2, 1 << 20), (3, (1 << 20) - 3)]


@pytest.mark.parametrize("b,v", TWO_LAUNCHES)
def test_every_form_of_two_launches(dev, b, v):
    """Random rows with all filters, ties that reach over the workgroups of a row, rows of one
    value (a workgroup's count at its largest), masks on either side, the largest at the end."""
    logits = _logits(b, v, dev, v + b)
    logits[0] = 0.5
    logits[1] = torch.randint(0, 3, (v,), device=dev, generator=torch.Generator(device=dev).manual_seed(v))
    if b > 2:
        logits[2, : v - 40000] = torch.finfo(torch.bfloat16).min
    if b > 8:
        logits[3, 40000:] = -math.inf
        logits[4, v - 1] = 90.0
        logits[5] = -1.0
        logits[5, ::7] = math.nan
        logits[6] = -250.0
        logits[6, 3::32768] = 1.0
        logits[7, v // 2] = 300.0  # (the second path)
    u = _uniform(b, dev, v)
    t = [0.0 if i == 9 else 0.5 + 0.1 * (i % 8) for i in range(b)]
    k = [v // 2 + 7, v // 3, 0, 50, 1000, v - 5, 30, 20][:b] + [[0, 1, 40, 5000][i % 4] for i in range(b - 8)]
    p = [[0.7, 0.95, 1.0, 0.3][i % 4] for i in range(b)]
    _check(dev, logits, u, t)
    _check(dev, logits, u, t, top_k=k)
    _check(dev, logits, u, t, top_p=p, top_k=k, min_p=[[0.0, 0.02, 0.001][i % 3] for i in range(b)])


def test_rows_far_apart_of_two_launches(dev):
    """Rows whose offsets pass 2^32 bytes, in workgroups of 32,768 tokens."""
    b, v, apart = 34, 250007, 1 << 26
    wide = torch.empty((b - 1) * apart + v, dtype=torch.bfloat16, device=dev)
    logits = wide.as_strided((b, v), (apart, 1))
    logits.normal_(std=3.0, generator=torch.Generator(device=dev).manual_seed(1))
    u = _uniform(b, dev, 2)
    _check(dev, logits, u, [0.8] * b, top_p=[0.95] * b, top_k=[100] * b, min_p=[0.01] * b)


def test_on_a_side_stream_and_two_samplers_at_once(dev):
    """A draw on a stream of its own, in order with what made its logits there; two samplers
    on two streams at once, eager and replayed: each the ids that it draws alone."""
    from minimal_inference_amd.sampling import Sampler

    b, v = 12, 152064
    made = [(_logits(b, v, dev, i), _uniform(b, dev, i)) for i in range(2)]
    samplers, want = [], []
    for logits, u in made:
        s = Sampler(dev, b, vocab=v)
        s.set_params([0.7] * b, [0.9] * b, top_k=[60] * b, min_p=[0.01] * b)
        samplers.append(s)
        want.append(s.draw(logits, u).tolist())
    f = lambda x: torch.tensor(x).double().item()  # noqa: E731
    assert want[0] == [draw_row(made[0][0][i].cpu(), made[0][1][i].item(), f(0.7), 60, f(0.9), f(0.01)) for i in range(b)]
    streams = [torch.cuda.Stream() for _ in made]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (s, stream, (logits, u)) in enumerate(zip(samplers, streams, made)):
            with torch.cuda.stream(stream):
                there = (logits + 1).sub_(1)  # (rounds: other logits, made on this stream)
                got[i].append((there, s.draw(there, u).clone(), s.draw(logits, u).clone()))
    torch.cuda.synchronize()
    for i, (s, (logits, u)) in enumerate(zip(samplers, made)):
        for there, moved, same in got[i]:
            assert same.tolist() == want[i]
            assert torch.equal(s.draw(there, u), moved)
    graphs, ids = [], []
    for s, stream, (logits, u) in zip(samplers, streams, made):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            ids.append(s.draw(logits, u))
        graphs.append(g)
    for _ in range(5):
        for t in ids:
            t.fill_(-1)
        torch.cuda.synchronize()
        for g, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                g.replay()
        torch.cuda.synchronize()
        assert [t.tolist() for t in ids] == want
