"""CPU: what the gated products' fp32 sums and the adapters' ends over them refuse before a launch."""

from __future__ import annotations

import ctypes

import pytest
import torch

FAKE = 1 << 32  # an aligned address that no refused call reads
SUMS, STEPS = 2, 3


def _lib():
    from minimal_inference_amd import _lib

    return _lib, _lib.load()


def test_names_agree_with_the_header():
    from pathlib import Path

    from minimal_inference_amd import _util

    header = (Path(__file__).resolve().parent.parent / "include" / "mi_amd.h").read_text()
    for name, value in (("MI_SILU", _util.SILU), ("MI_SILU_SUMS", _util.SILU_SUMS), ("MI_SILU_STEPS", _util.SILU_STEPS)):
        assert f"#define {name} {value} " in header


LINEAR8 = dict(x=FAKE, xs=64, xsc=FAKE + (1 << 20), xss=16, w=FAKE + (1 << 21), ws=64, wsc=FAKE + (1 << 22), wss=16, bias=None,
               out=FAKE + (1 << 23), os=64, osc=None, oss=0, rows=4, n=32, k=64, silu=SUMS, work=None, bytes=0)
LINEAR4 = dict(x=FAKE, xs=64, xsc=None, w=FAKE + (1 << 21), wsc=FAKE + (1 << 22), bias=None, out=FAKE + (1 << 23), os=64, rows=4, n=32,
               k=64, silu=SUMS, work=None, bytes=0)
COMMON = [{"n": 30, "os": 60}, {"os": 60}, {"os": 66}, {"out": FAKE + (1 << 23) + 8}, {"bias": FAKE}, {"out": FAKE + 64 * 3 + 48},
          {"out": FAKE + (1 << 21) - 16}, {"out": FAKE + (1 << 21) - 3 * 256 - 240}]


@pytest.mark.parametrize("change", COMMON + [{"osc": FAKE + (1 << 24), "oss": 1}])
def test_linear_mxfp8_refuses(change):
    mod, lib = _lib()
    assert lib.mi_linear_mxfp8(*(LINEAR8 | change).values(), None) == mod.MI_ERR_INVALID
    assert mod.last_error().startswith("linear_mxfp8")


@pytest.mark.parametrize("change", COMMON)
def test_linear_mxfp4_refuses(change):
    mod, lib = _lib()
    assert lib.mi_linear_mxfp4(*(LINEAR4 | change).values(), None) == mod.MI_ERR_INVALID
    assert mod.last_error().startswith("linear_mxfp4")


ADAPT = dict(y=FAKE, ys=64, x=FAKE + (1 << 20), xs=96, xsc=None, xss=0, a=FAKE + (1 << 21), b=FAKE + (1 << 22), scale=FAKE + (1 << 23),
             slots=3, k=96, rank=24, pieces=(32, 32), n_pieces=2, out=FAKE + (1 << 24), os=32, osc=None, oss=0, plan=FAKE + (1 << 25), rows=4,
             silu=SUMS, work=FAKE + (1 << 26), bytes=1 << 24)


@pytest.mark.parametrize("change", [
    {"ys": 66}, {"y": FAKE + 8}, {"pieces": (32, 16)}, {"n_pieces": 1, "pieces": (64,)}, {"os": 24},
    {"out": FAKE + 3 * 256 + 240}, {"osc": FAKE + 3 * 256 + 255, "oss": 1, "os": 64}, {"work": FAKE + 3 * 256 + 240},
    {"silu": STEPS, "osc": FAKE + (1 << 27), "oss": 1}, {"silu": STEPS, "ys": 68}, {"silu": STEPS, "out": FAKE}, {"silu": STEPS, "pieces": (48, 16)}])
def test_add_adapters_refuses(change):
    mod, lib = _lib()
    a = ADAPT | change
    held = (ctypes.c_int32 * len(a["pieces"]))(*a["pieces"])
    a["pieces"] = ctypes.addressof(held)
    assert lib.mi_add_adapters(*a.values(), None) == mod.MI_ERR_INVALID
    assert mod.last_error().startswith("add_adapters")


def test_python_refusals_on_the_cpu():
    from minimal_inference_amd.adapters import add_adapters_silu
    from minimal_inference_amd.mxfp4 import gate_up_mxfp4
    from minimal_inference_amd.mxfp8 import MXFP8, gate_up_mxfp8

    m = MXFP8(4, 64, "cpu")
    for call in (lambda: gate_up_mxfp8(m, MXFP8(5, 64, "cpu")), lambda: gate_up_mxfp8(m, MXFP8(12, 64, "cpu")),
                 lambda: gate_up_mxfp8(m, MXFP8(16, 96, "cpu")), lambda: gate_up_mxfp8(m, MXFP8(16, 64, "cpu"), out=torch.zeros(4, 16)),
                 lambda: add_adapters_silu(torch.zeros(4, 64), None, None, None, quantize=True, stepwise=True),
                 lambda: add_adapters_silu(torch.zeros(4, 64), None, None, None)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        gate_up_mxfp4(torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(8, 64))


@pytest.mark.gpu
def test_refused_on_the_gpu(dev):
    from minimal_inference_amd.adapters import AdapterPlan, Adapters, add_adapters, add_adapters_silu
    from minimal_inference_amd.mxfp4 import gate_up_mxfp4, quantize_mxfp4
    from minimal_inference_amd.mxfp8 import gate_up_mxfp8, quantize_mxfp8

    x = torch.randn(5, 64, device=dev).to(torch.bfloat16)
    w = torch.randn(64, 64, device=dev).to(torch.bfloat16)
    w8, w4, m = quantize_mxfp8(w), quantize_mxfp4(w), quantize_mxfp8(x)
    ad, plan = Adapters.empty(2, 64, [32, 32], 8, dev), AdapterPlan(5, 2, dev)
    plan.plan(torch.zeros(5, dtype=torch.int32, device=dev))
    y = gate_up_mxfp8(m, w8)
    assert y.shape == (5, 64) and y.dtype == torch.float32
    assert gate_up_mxfp8(quantize_mxfp8(x[:0]), w8).shape == (0, 64) and gate_up_mxfp4(x[:0], w4).shape == (0, 64)
    for bad in (torch.empty(5, 32, device=dev), torch.empty(5, 64, device=dev, dtype=torch.bfloat16), torch.empty(5, 65, device=dev)[:, 1:],
                torch.empty(5, 128, device=dev)[:, ::2], torch.empty(5, 64, device=dev, requires_grad=True)):
        for call in (lambda: gate_up_mxfp8(m, w8, out=bad), lambda: gate_up_mxfp4(x, w4, out=bad)):
            with pytest.raises(ValueError):
                call()
    for call in (lambda: add_adapters_silu(y, x, ad, plan, stepwise=True), lambda: add_adapters(y, x, ad, plan),
                 lambda: add_adapters_silu(y.double(), x, ad, plan), lambda: add_adapters_silu(y[:, :32], x, ad, plan),
                 lambda: add_adapters_silu(y.clone().requires_grad_(), x, ad, plan), lambda: add_adapters_silu(y[:, ::2], x, ad, plan)):
        with pytest.raises((ValueError, RuntimeError)):
            call()
