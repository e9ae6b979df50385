"""GPU: the filtered draw from given uniform numbers against the same draw in 64 bits.

Ids are equal: the kernels count values and sum in 64 bits, so a draw falls on the other
side of a border only within some 2^-50 of it.
"""

from __future__ import annotations

import math

import pytest
import torch

from oracle.draw import draw_row

pytestmark = pytest.mark.gpu


def _sampler(dev, batch, vocab, temperature, top_p=None, top_k=None, min_p=None):
    from minimal_inference_amd.sampling import Sampler

    s = Sampler(dev, batch, vocab=vocab)
    s.set_params(temperature, top_p, top_k=top_k, min_p=min_p)
    return s


def _check(dev, logits, u, temperature, top_p=None, top_k=None, min_p=None):
    b, v = logits.shape
    got = _sampler(dev, b, v, temperature, top_p, top_k, min_p).draw(logits, u).tolist()
    host, uh = logits.cpu(), u.cpu().double().tolist()
    f32 = lambda x: torch.tensor(x, dtype=torch.float32).double().tolist()  # noqa: E731
    t, p, m = f32(temperature), f32(top_p or [1.0] * b), f32(min_p or [0.0] * b)
    k = top_k or [0] * b
    want = [draw_row(host[i], uh[i], t[i], k[i], p[i], m[i]) for i in range(b)]
    assert got == want


def _uniform(n, dev, seed):
    return torch.rand(n, device=dev, generator=torch.Generator(device=dev).manual_seed(seed))


def _logits(b, v, dev, seed, spread=3.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(b, v, device=dev, generator=g) * spread).to(torch.bfloat16)


@pytest.mark.parametrize("vocab", [1, 2, 7, 100, 1023, 4097, 32767, 32768, 32769, 65541, 151929, 152064])
def test_every_filter(dev, vocab):
    """Each filter alone and together, in one batch, over vocabularies of one token, odd
    ones (rows at any alignment) and several chunks."""
    b = 24
    t = [0.0 if i == 5 else 0.3 + 0.15 * (i % 9) for i in range(b)]
    k = [[0, 1, 2, 50, 1000, 40000][i % 6] for i in range(b)]
    p = [[1.0, 0.0, 0.1, 0.5, 0.9, 0.999, 1.5][i % 7] for i in range(b)]
    m = [[0.0, 0.001, 0.05, 0.5, 1.0, 2.0][(i // 2) % 6] for i in range(b)]
    logits, u = _logits(b, vocab, dev, vocab), _uniform(b, dev, 1)
    off = [0.0] * b
    _check(dev, logits, u, t)
    _check(dev, logits, u, t, top_k=k)
    _check(dev, logits, u, t, top_p=p)
    _check(dev, logits, u, t, min_p=m)
    _check(dev, logits, u, t, top_p=p, top_k=k, min_p=m)
    _check(dev, logits, u, off)


@pytest.mark.parametrize("b,v", [(12, 5000), (12, 8192), (12, 8193), (12, 16384), (32, 16385), (36, 32761), (36, 32768), (31, 32768)])
def test_rows_of_one_chunk_and_beside_them(dev, b, v):
    """Short rows, which one launch counts and draws, up to the sizes where two begin:
    ties cut inside a value, masks, NaN, infinities, values outside the counted range,
    greedy rows."""
    logits = _logits(b, v, dev, v + b)
    logits[0] = 0
    logits[1] = torch.randint(0, 3, (v,), device=dev, generator=torch.Generator(device=dev).manual_seed(1))
    logits[2, 17:] = -math.inf
    logits[3, 5:v - 3] = torch.finfo(torch.bfloat16).min
    logits[4, ::2] = math.nan
    logits[5, v // 2] = math.inf
    logits[6] *= 300
    logits[7, 9] = 2.0 ** -40
    logits[8] = -math.inf
    logits[9] = math.nan
    u = _uniform(b, dev, v)
    t = [0.0 if i in (10, 11) else 0.4 + 0.1 * (i % 9) for i in range(b)]
    _check(dev, logits, u, t)
    _check(dev, logits, u, t, top_k=[v // 3, 7, 3, 50][:4] * (b // 4) + [1] * (b % 4))
    _check(dev, logits, u, t, top_p=[0.3, 0.9, 1.0] * (b // 3) + [0.5] * (b % 3), min_p=[0.0, 0.02] * (b // 2) + [0.1] * (b % 2))
    _check(dev, logits, u, [50.0] * b, top_k=[1000] * b, top_p=[0.7] * b, min_p=[0.001] * b)


def test_ties_go_to_the_lowest_index(dev):
    """Rows of one value and of three, cut inside a value by top-k and by top-p, over
    several chunks."""
    v = 70000
    logits = torch.zeros(12, v, device=dev, dtype=torch.bfloat16)
    logits[6:] = torch.randint(0, 3, (6, v), device=dev, generator=torch.Generator(device=dev).manual_seed(0))
    u = _uniform(12, dev, 2)
    t = [1.0, 0.5] * 6
    _check(dev, logits, u, t, top_k=[1, 2, 33000, 69999, 70000, 5] * 2)
    _check(dev, logits, u, t, top_p=[0.5, 0.25, 0.75, 0.9, 0.001, 1.0] * 2)
    _check(dev, logits, u, t, top_p=[0.5, 0.25, 0.75, 0.9, 0.001, 1.0] * 2, top_k=[40000] * 12, min_p=[0.3] * 12)


def test_uniforms_at_their_ends(dev):
    """u = 0 draws the first kept index and the largest float below 1 the last of weight."""
    logits = _logits(6, 40000, dev, 9)
    top = 1.0 - 2.0 ** -24
    u = torch.tensor([0.0, top, 0.0, top, 0.0, top], device=dev)
    t = [0.7, 0.7, 1.0, 1.0, 5.0, 5.0]
    _check(dev, logits, u, t)
    _check(dev, logits, u, t, top_k=[3] * 6)
    _check(dev, logits, u, t, top_p=[0.9] * 6, min_p=[0.01] * 6)


def test_masked_and_non_finite_rows(dev):
    """-inf and the type's lowest value as masks, rows with one token or none left,
    NaN (never drawn, highest for greedy rows), +inf (takes all weight)."""
    v = 33000
    logits = _logits(14, v, dev, 4)
    lowest = torch.finfo(torch.bfloat16).min
    logits[0, 10:] = -math.inf
    logits[1, :32990] = lowest
    logits[2] = -math.inf
    logits[3] = lowest
    logits[4] = math.nan
    logits[5, 100] = math.nan
    logits[6, [5, 900, 32999]] = math.inf
    logits[7, :] = -math.inf
    logits[7, 32998] = 2.0
    logits[8, 3], logits[8, 4:] = math.nan, -math.inf
    logits[9, 7] = math.nan  # greedy
    logits[10] = -math.inf   # greedy
    logits[11, 0] = -math.inf
    logits[12] = -1000.0
    logits[12, 77], logits[12, 78] = -999.0, -996.0
    t = [0.8] * 9 + [0.0, 0.0, 1.0, 1.0, 1.0]
    u = _uniform(14, dev, 5)
    _check(dev, logits, u, t)
    _check(dev, logits, u, t, top_k=[20] * 14, top_p=[0.9] * 14, min_p=[0.02] * 14)


@pytest.mark.parametrize("scale", [1e-10, 1e-3, 40.0, 3e3, 1e30])
def test_values_outside_the_counted_range(dev, scale):
    """Rows of tiny and of huge logits take the second path: the same draws."""
    b, v = 8, 33500
    logits = _logits(b, v, dev, 6, spread=scale)
    u = _uniform(b, dev, 7)
    t = [scale * (0.3 + 0.1 * i) for i in range(b)]
    _check(dev, logits, u, t)
    _check(dev, logits, u, t, top_k=[0, 1, 5, 40, 1000, 33499, 33500, 20000])
    _check(dev, logits, u, t, top_p=[0.1, 0.5, 0.9, 0.99, 0.0, 1.0, 0.7, 0.3], min_p=[0.0, 0.1] * 4)
    _check(dev, logits, u, t, top_k=[50] * b, top_p=[0.9] * b, min_p=[0.01] * b)


def test_low_values_at_every_temperature(dev):
    """Values on either side of -2^8 and the type's lowest as masks, at temperatures at
    which the ones weigh something and the others do not."""
    v = 20000
    logits = _logits(10, v, dev, 21)
    logits[:, 100:15000] = torch.finfo(torch.bfloat16).min
    logits[2:, ::3] -= 257
    logits[4:6, 1::2] = -256
    logits[6:8] -= 400
    logits[8, 1:] = -255
    u = _uniform(10, dev, 22)
    for scale in (1.0, 6.0, 100.0):
        t = [scale * (0.5 + 0.1 * i) for i in range(10)]
        _check(dev, logits, u, t)
        _check(dev, logits, u, t, top_k=[0, 6000, 40, 15000, 1, 9000, 50, 0, 3, 19999], top_p=[0.95] * 10)


def test_extreme_temperatures(dev):
    logits, u = _logits(6, 5000, dev, 8), _uniform(6, dev, 8)
    t = [1e-30, 1e-3, 1e3, 1e30, math.inf, math.nan]
    _check(dev, logits, u, t)
    _check(dev, logits, u, t, top_k=[7] * 6, top_p=[0.6] * 6)


def test_the_draws_follow_the_weights(dev):
    """Equally spaced u draw each kept token as often as its weight says, to one draw."""
    n, v = 4000, 300
    row = _logits(1, v, dev, 3)
    logits = row.expand(n, v).contiguous()
    u = (torch.arange(n, device=dev, dtype=torch.float32) + 0.5) / n
    ids = _sampler(dev, n, v, [0.9] * n, [1.0] * n, [40] * n, [0.0] * n).draw(logits, u)
    l = row[0].double()
    keep = torch.argsort(l, descending=True, stable=True)[:40]
    p = torch.zeros(v, device=dev, dtype=torch.float64)
    p[keep] = torch.softmax(l[keep] / torch.tensor(0.9).double().item(), 0)
    share = torch.bincount(ids, minlength=v).double()
    assert bool(((share - n * p).abs() <= 1.0).all())


def test_strides_partial_batches_and_replays(dev):
    """Rows of a wider buffer, n below the batch, an out of the caller's with what lies
    behind it left as it was, another order of calls on one sampler, and a captured draw
    replayed on new logits, numbers and parameters."""
    b, v = 5, 40001
    wide = _logits(b, v + 3, dev, 11)
    logits = wide[:, 1:1 + v]
    u = _uniform(8, dev, 12)
    s = _sampler(dev, 8, v, [0.9] * b, [0.9] * b, [30] * b, [0.01] * b)
    out = torch.full((8,), -7, dtype=torch.int64, device=dev)
    got = s.draw(logits, u, 3, out=out)
    f = lambda x: torch.tensor(x).double().item()  # noqa: E731
    want = [draw_row(logits[i].cpu(), u[i].item(), f(0.9), 30, f(0.9), f(0.01)) for i in range(b)]
    assert got.tolist() == want[:3] and out[3:].tolist() == [-7] * 5
    assert s.draw(logits[:, None, :], u).tolist() == want
    s.draw(_logits(8, 100, dev, 1), u)
    assert s.draw(logits, u).tolist() == want
    graph = torch.cuda.CUDAGraph()
    still, numbers = logits.contiguous(), u.clone()
    with torch.cuda.graph(graph):
        ids = s.draw(still, numbers)
    for seed in range(4):
        still.copy_(_logits(b, v, dev, 20 + seed))
        numbers.copy_(_uniform(8, dev, 30 + seed))
        s.set_params([0.5 + 0.2 * seed] * b, [0.95] * b, top_k=[seed * 10] * b, min_p=[0.0] * b)
        graph.replay()
        held = ids.tolist()
        t, p = f(0.5 + 0.2 * seed), f(0.95)
        assert held == [draw_row(still[i].cpu(), numbers[i].item(), t, seed * 10, p) for i in range(b)]
        assert s.draw(still, numbers).tolist() == held


def test_sample_batch_takes_the_filters(dev):
    """sample_batch / sample: with given numbers the oracle's ids; top-k of one is
    greedy; a call without them after one with them is the plain sampler again."""
    from minimal_inference_amd.sampling import _sampler_for, sample, sample_batch

    b, v = 4, 32768
    logits = _logits(b, v, dev, 13).view(b, 1, v)
    u = _uniform(b, dev, 14)
    f = lambda x: torch.tensor(x).double().item()  # noqa: E731
    got = sample_batch(logits, [0.7] * b, [0.9] * b, top_k=[40] * b, min_p=[0.05] * b, uniforms=u)
    assert got == [draw_row(logits[i, 0].cpu(), u[i].item(), f(0.7), 40, f(0.9), f(0.05)) for i in range(b)]
    greedy = logits[:, 0].float().argmax(-1).tolist()
    assert sample_batch(logits, [1.0] * b, top_k=[1] * b) == greedy
    assert sample(logits[:1], 1.0, min_p=1.0, uniforms=u[:1]) == greedy[0]
    s = _sampler_for(dev, b)
    s.rng_offset.zero_()
    first = sample_batch(logits, [0.7] * b, [0.9] * b)
    s.rng_offset.zero_()
    assert sample_batch(logits, [0.7] * b, [0.9] * b) == first
    assert s.top_k.tolist() == [0] * b and s.min_p.tolist() == [0.0] * b


def test_refused(dev):
    from minimal_inference_amd.sampling import Sampler, sample_batch

    s = Sampler(dev, 4, vocab=100)
    logits, u = _logits(4, 100, dev, 1), _uniform(4, dev, 1)
    for bad in [lambda: s.draw(logits.float(), u), lambda: s.draw(logits, u.double()), lambda: s.draw(logits, u[:3]),
                lambda: s.draw(logits, u, 5), lambda: s.draw(logits, u, -1), lambda: s.draw(logits[:, ::2], u),
                lambda: s.draw(logits, u.cpu()), lambda: s.draw(logits, u, out=torch.zeros(4, device=dev)),
                lambda: s.draw(logits, u, out=torch.zeros(3, dtype=torch.int64, device=dev)),
                lambda: s.draw(logits.cpu(), u), lambda: s.draw(_logits(5, 100, dev, 1), _uniform(5, dev, 1)),
                lambda: sample_batch(logits[:, None], [1.0] * 4, top_k=[1])]:
        with pytest.raises(ValueError):
            bad()
    assert s.draw(logits[:0], u).tolist() == []
    with pytest.raises(ValueError):
        s.draw(torch.zeros(1, (1 << 20) + 1, dtype=torch.bfloat16, device=dev), u)
