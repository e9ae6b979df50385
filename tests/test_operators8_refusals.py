"""CPU: what the 8-bit and adapter operators refuse before a launch, their sizes, the oracle's hand-made
cases, and the server's adapter names."""

from __future__ import annotations

import ctypes

import pytest
import torch

FAKE = 1 << 32  # an aligned address that no refused call reads


def _lib():
    from minimal_inference_amd import _lib

    return _lib, _lib.load()


def _refused(entry, args, what, code=None):
    mod, lib = _lib()
    assert getattr(lib, entry)(*args.values(), None) == (mod.MI_ERR_INVALID if code is None else code)
    assert mod.last_error().startswith(what)


@pytest.mark.parametrize("entry", ["mi_mxfp8_quantize", "mi_mxfp8_dequantize"])
@pytest.mark.parametrize("change", [
    {"rows": -1}, {"rows": (1 << 31) + 1}, {"cols": 0}, {"cols": 48}, {"cols": (1 << 20) + 32}, {"x": None}, {"codes": None},
    {"scales": None}, {"x": FAKE + 8}, {"xs": 68}, {"xs": 56}, {"codes": FAKE + (1 << 24) + 8}, {"cs": 72}, {"cs": 48}, {"ss": 1},
    {"codes": FAKE}, {"codes": FAKE + 384 + 48}, {"scales": FAKE + 128 * 3 + 127}, {"scales": FAKE + (1 << 24) + 64 * 3 + 63},
    {"rows": 1 << 31, "codes": FAKE + 128}])
def test_rows_refuse(entry, change):
    """Four rows of 64 values: x at 0, codes at 2^24, scales at 2^25."""
    a = dict(x=FAKE, xs=64, codes=FAKE + (1 << 24), cs=64, scales=FAKE + (1 << 25), ss=2, rows=4, cols=64) | change
    if entry == "mi_mxfp8_dequantize":
        a = dict(codes=a["codes"], cs=a["cs"], scales=a["scales"], ss=a["ss"], x=a["x"], xs=a["xs"], rows=a["rows"], cols=a["cols"])
    _refused(entry, a, entry[3:])


@pytest.mark.parametrize("change", [
    {"rows": -1}, {"rows": (1 << 22) + 1}, {"hidden": 0}, {"hidden": 48}, {"hidden": 16416}, {"x": None}, {"weight": None},
    {"codes": None}, {"scales": None}, {"x": FAKE + 8}, {"xs": 68}, {"d": FAKE + 8}, {"ds": 4}, {"weight": FAKE + 8}, {"xo": FAKE + 2},
    {"xos": 56}, {"cs": 56}, {"cs": 48}, {"ss": 1},
    {"xo": FAKE + 16}, {"xo": FAKE + 128}, {"xo": FAKE + (1 << 24) + 128}, {"codes": FAKE}, {"codes": FAKE + 16}, {"scales": FAKE + 130},
    {"codes": FAKE + (1 << 26) + 128}, {"scales": FAKE + (1 << 27) + 255}, {"codes": FAKE + (1 << 25) + 112}, {"scales": FAKE + (1 << 25)},
    {"rows": 1, "codes": FAKE + (1 << 25)}, {"xs": 0, "xo": FAKE}])
def test_norm_refuses(change):
    """Four rows of 64 values: x at 0, delta at 2^24, weight at 2^25, x_out at 2^26, codes at 2^27, scales at 2^28."""
    a = dict(x=FAKE, xs=64, d=FAKE + (1 << 24), ds=64, weight=FAKE + (1 << 25), xo=FAKE + (1 << 26), xos=64, codes=FAKE + (1 << 27),
             cs=64, scales=FAKE + (1 << 28), ss=2, rows=4, hidden=64, eps=1e-6) | change
    _refused("mi_add_rms_norm_mxfp8", a, "add_rms_norm_mxfp8")


LINEAR = dict(x=FAKE, xs=64, xsc=FAKE + (1 << 20), xss=16, w=FAKE + (1 << 21), ws=64, wsc=FAKE + (1 << 22), wss=16, bias=None,
              out=FAKE + (1 << 23), os=32, osc=None, oss=0, rows=4, n=32, k=64, silu=0, work=None, bytes=0)


@pytest.mark.parametrize("change", [
    {"rows": -1}, {"rows": (1 << 22) + 1}, {"n": 0}, {"n": (1 << 24) + 1}, {"k": 0}, {"k": 48}, {"k": (1 << 20) + 32}, {"x": None},
    {"xsc": None}, {"w": None}, {"wsc": None}, {"out": None}, {"x": FAKE + 8}, {"xsc": FAKE + 4}, {"w": FAKE + 8}, {"wsc": FAKE + 8},
    {"xs": 72}, {"xs": 48}, {"xss": 8}, {"xss": 0}, {"ws": 48}, {"wss": 24}, {"ws": (1 << 22) + 16}, {"xss": (1 << 22) + 16},
    {"out": FAKE + (1 << 23) + 1}, {"bias": FAKE + 1}, {"os": 31}, {"silu": 1, "bias": FAKE}, {"work": FAKE + 8, "bytes": 64},
    {"osc": FAKE + (1 << 24), "oss": 1}, {"silu": 1, "n": 16, "os": 16, "osc": FAKE + (1 << 24), "oss": 1},
    {"silu": 1, "osc": FAKE + (1 << 24), "oss": 0}, {"silu": 1, "osc": FAKE + (1 << 24), "oss": 1, "out": FAKE + (1 << 23) + 8},
    {"silu": 1, "osc": FAKE + (1 << 24), "oss": 1, "os": 40},
    {"out": FAKE}, {"out": FAKE + 64 * 3 + 62}, {"out": FAKE + (1 << 20)}, {"out": FAKE + (1 << 21) + 64 * 31 + 62},
    {"out": FAKE + (1 << 22) - 254}, {"bias": FAKE + (1 << 23) + 254}, {"silu": 1, "out": FAKE + (1 << 21) + 64 * 63 + 62},
    {"silu": 1, "osc": FAKE + (1 << 23) + 32 * 3 + 31, "oss": 1}, {"silu": 1, "osc": FAKE + 63, "oss": 1}])
def test_linear_refuses(change):
    _refused("mi_linear_mxfp8", LINEAR | change, "linear_mxfp8")


def test_linear_takes_no_rows():
    mod, lib = _lib()
    assert lib.mi_linear_mxfp8(*(LINEAR | {"rows": 0, "x": None}).values(), None) == mod.MI_OK
    assert lib.mi_linear_mxfp8_workspace_size(64, 32, 64, 0) == 0  # few rows take none
    for bad in ((0, 32, 64, 0), (1 << 23, 32, 64, 0), (100, 0, 64, 0), (100, 32, 48, 0)):
        assert lib.mi_linear_mxfp8_workspace_size(*bad) == 0


def _pieces(*n):
    return (ctypes.c_int32 * len(n))(*n)


@pytest.mark.parametrize("change", [
    {"rows": -1}, {"rows": (1 << 22) + 1}, {"slots": 0}, {"slots": 1024}, {"plan": None}, {"slot": None}, {"plan": FAKE + 8},
    {"slot": FAKE + 2}, {"slot": FAKE + (1 << 24) + 64}])
def test_plan_refuses(change):
    a = dict(plan=FAKE + (1 << 24), bytes=1 << 20, slot=FAKE, rows=40, slots=3) | change
    _refused("mi_adapter_plan", a, "adapter_plan")


def test_plan_sizes():
    mod, lib = _lib()
    size = lib.mi_adapter_plan_size
    assert size(0, 1) > 0 and size(1, 1023) >= 16 + 16 + 4
    for bad in ((-1, 1), ((1 << 22) + 1, 1), (5, 0), (5, 1024)):
        assert size(*bad) == 0
    for slots in (1, 3, 100):  # room for every smaller batch
        sizes = [size(r, slots) for r in range(0, 1300)]
        assert sizes == sorted(sizes)
    _refused("mi_adapter_plan", dict(plan=FAKE, bytes=size(40, 3) - 1, slot=FAKE + (1 << 20), rows=40, slots=3), "adapter_plan",
             mod.MI_ERR_WORKSPACE)


ADAPT = dict(y=FAKE, ys=64, x=FAKE + (1 << 20), xs=96, xsc=None, xss=0, a=FAKE + (1 << 21), b=FAKE + (1 << 22), scale=FAKE + (1 << 23),
             slots=3, k=96, rank=24, pieces=(48, 16), n_pieces=2, out=FAKE + (1 << 24), os=64, osc=None, oss=0, plan=FAKE + (1 << 25), rows=4,
             silu=0, work=FAKE + (1 << 26), bytes=1 << 24)


@pytest.mark.parametrize("change", [
    {"rows": -1}, {"slots": 0}, {"slots": 1024}, {"k": 80}, {"k": 0}, {"k": (1 << 20) + 32}, {"rank": 0}, {"rank": 12}, {"rank": 136},
    {"n_pieces": 0}, {"n_pieces": 9, "pieces": (16,) * 9}, {"pieces": (48, 8)}, {"pieces": (0, 64)}, {"pieces": (-16, 80)},
    {"pieces": ((1 << 20) + 16, 16)}, {"pieces": None}, {"y": None}, {"x": None}, {"a": None}, {"b": None}, {"scale": None}, {"out": None},
    {"plan": None}, {"work": None}, {"y": FAKE + 8}, {"x": FAKE + 8}, {"a": FAKE + 8}, {"b": FAKE + 8}, {"scale": FAKE + 2}, {"ys": 68},
    {"os": 68}, {"os": 56}, {"xs": 100}, {"xs": -96}, {"xsc": FAKE + 8, "xss": 16}, {"xsc": FAKE + (1 << 19), "xss": 8},
    {"xsc": FAKE + (1 << 19), "xss": 0}, {"xsc": FAKE + (1 << 19), "xss": 16, "xs": 104},
    {"out": FAKE + 16}, {"out": FAKE, "os": 72}, {"out": FAKE + (1 << 20)}, {"out": FAKE + (1 << 21) + 3 * 48 * 96 * 2 - 16},
    {"out": FAKE + (1 << 22) + 3 * 64 * 24 * 2 - 16}, {"out": FAKE + (1 << 25)}, {"out": FAKE + (1 << 26)}, {"scale": FAKE + (1 << 24) + 8},
    {"silu": 1}, {"silu": 1, "pieces": (32, 16)}, {"silu": 1, "n_pieces": 1, "pieces": (64,)}, {"osc": FAKE + (1 << 27), "oss": 1},
    {"silu": 1, "pieces": (16, 16), "osc": FAKE + (1 << 27), "oss": 1}, {"silu": 1, "pieces": (32, 32), "osc": FAKE + (1 << 27)},
    {"silu": 1, "pieces": (32, 32), "os": 24}, {"silu": 1, "pieces": (32, 32), "os": 40, "osc": FAKE + (1 << 27), "oss": 1},
    {"silu": 1, "pieces": (32, 32), "out": FAKE}, {"silu": 1, "pieces": (32, 32), "out": FAKE + 64},
    {"silu": 1, "pieces": (32, 32), "osc": FAKE + (1 << 24) + 31, "oss": 1}, {"silu": 1, "pieces": (32, 32), "osc": FAKE + 9, "oss": 1}])
def test_add_adapters_refuses(change):
    a = ADAPT | change
    held = None if a["pieces"] is None else _pieces(*a["pieces"])
    a["pieces"] = None if held is None else ctypes.addressof(held)
    _refused("mi_add_adapters", a, "add_adapters")


def test_add_adapters_workspace():
    mod, lib = _lib()
    assert lib.mi_add_adapters_workspace_size(4, 3, 96, 24, 2, 64, 0) > 0  # (two launches)
    assert lib.mi_add_adapters_workspace_size(4, 3, 96, 16, 2, 64, 0) == 0  # (one)
    assert lib.mi_add_adapters_workspace_size(4, 3, 96, 16, 2, 64, 1) > 0
    held = _pieces(48, 16)
    _refused("mi_add_adapters", ADAPT | {"pieces": ctypes.addressof(held), "bytes": 0}, "add_adapters", mod.MI_ERR_WORKSPACE)
    assert lib.mi_add_adapters(*(ADAPT | {"pieces": ctypes.addressof(held), "rows": 0, "y": None}).values(), None) == mod.MI_OK
    for bad in ((-1, 3, 96, 24, 2, 64, 0), (4, 0, 96, 24, 2, 64, 0), (4, 3, 80, 24, 2, 64, 0), (4, 3, 96, 12, 2, 64, 0),
                (4, 3, 96, 24, 9, 64, 0), (0, 3, 96, 24, 2, 64, 0)):
        assert lib.mi_add_adapters_workspace_size(*bad) == 0


def test_python_refusals_on_the_cpu():
    """What needs no GPU to be told."""
    from minimal_inference_amd.adapters import AdapterPlan, Adapters, add_adapters
    from minimal_inference_amd.mxfp8 import MXFP8, add_rms_norm_mxfp8, linear_mxfp8, linear_silu_mxfp8, quantize_mxfp8

    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    w = torch.zeros(64, dtype=torch.bfloat16)
    for call in (lambda: quantize_mxfp8(x), lambda: add_rms_norm_mxfp8(x, None, w, 1e-6), lambda: MXFP8(-1, 64, "cpu"),
                 lambda: MXFP8(4, 48, "cpu"), lambda: MXFP8(4, 0, "cpu"), lambda: MXFP8(4, (1 << 20) + 32, "cpu"),
                 lambda: MXFP8.from_codes(torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)),
                 lambda: add_rms_norm_mxfp8(torch.zeros(4, 16416, dtype=torch.bfloat16), None, w, 1e-6),
                 lambda: add_rms_norm_mxfp8(torch.zeros(64, dtype=torch.bfloat16), None, w, 1e-6),
                 lambda: AdapterPlan(4, 0, "cpu"), lambda: AdapterPlan(-1, 4, "cpu"), lambda: AdapterPlan(4, 1024, "cpu"),
                 lambda: Adapters.empty(2, 80, [16], 8, "cpu"), lambda: Adapters.empty(2, 64, [16], 8, "cpu"),
                 lambda: Adapters.empty(2, 64, [], 8, "cpu"), lambda: Adapters.empty(2, 64, [8], 8, "cpu"),
                 lambda: Adapters.empty(2, 64, [16] * 9, 8, "cpu"), lambda: Adapters.empty(2, 64, [16], 4, "cpu")):
        with pytest.raises(ValueError):
            call()
    m, v = MXFP8(4, 64, "cpu"), MXFP8(6, 64, "cpu")
    for call in (lambda: linear_mxfp8(x, m), lambda: linear_mxfp8(m, x), lambda: add_adapters(None, x, None, None)):
        with pytest.raises((TypeError, AttributeError)):
            call()
    for call in (lambda: linear_silu_mxfp8(m, MXFP8(5, 64, "cpu")), lambda: linear_mxfp8(m, MXFP8(6, 96, "cpu")),
                 lambda: linear_silu_mxfp8(m, v, quantize=True), lambda: linear_mxfp8(m, v, w[:6]),
                 lambda: linear_mxfp8(m, v, out=x)):
        with pytest.raises(ValueError):
            call()


def test_matrix_views():
    """Codes and scales are views of one buffer; scale rows are padded to whole 16 bytes."""
    from minimal_inference_amd.mxfp8 import MXFP8

    for cols, stride in ((32, 16), (512, 16), (544, 32), (4096, 128)):
        m = MXFP8(5, cols, "cpu")
        assert m.shape == (5, cols) and m.scales_stride == stride and m.nbytes == 5 * (cols + stride) == m.anchor.numel()
        assert m.codes.dtype == torch.float8_e4m3fn and m.codes.data_ptr() == m.codes_ptr and m.codes.stride(0) == m.codes_stride
        assert m.scales.shape == (5, cols // 32) and m.scales.data_ptr() == m.scales_ptr and m.scales.stride(0) == stride


def test_oracle_quantisation():
    """By hand: a maximum of 448 and above it, ties, the least values, zeros, infinities."""
    from oracle import mxfp8 as om8

    row = torch.zeros(1, 32, dtype=torch.float64)
    for top, byte in ((448.0, 127), (448.0000001, 128), (449.0, 128), (224.0, 126), (1.0, 119), (2.0 ** -119, 0), (2.0 ** -140, 0), (0.0, 0)):
        row[0, 3] = top
        assert int(om8.quantize(row)[1][0, 0]) == byte, top
    row[0, 0], row[0, 3] = 448.0, 17.0  # unit 1: halfway between 16 (even) and 18
    row[0, 4], row[0, 5], row[0, 6], row[0, 7] = 19.0, -2.0 ** -10, 2.0 ** -10 + 1e-9, -0.0
    codes, scales = om8.quantize(row)
    assert [float(v) for v in om8.values(codes, scales)[0, 3:8]] == [16.0, 20.0, 0.0, 2.0 ** -9, 0.0]
    assert codes[0, 5] == 128 and codes[0, 7] == 128
    row[0, 9] = float("inf")
    codes, scales = om8.quantize(row)
    assert int(scales[0, 0]) == 255 and not bool(codes.any()) and bool(om8.values(codes, scales).isnan().all())


def test_server_names_adapters():
    """A request's model picks an adapter; unknown names get none, as before."""
    from fastapi.testclient import TestClient

    from minimal_inference_amd.server import create_app
    from minimal_inference_amd.tokenizer import SyntheticTokenizer
    from tests.test_server import EOS, VOCAB, FakeScheduler

    sch = FakeScheduler([65, 66, EOS])
    app = create_app(sch, SyntheticTokenizer(VOCAB), "base", {EOS}, {"one": 0, "two": 1})
    with TestClient(app) as c:
        assert [m["id"] for m in c.get("/v1/models").json()["data"]] == ["base", "one", "two"]
        for name in ("two", "one", "base", "other", ""):
            r = c.post("/v1/chat/completions", json={"model": name, "messages": [{"role": "user", "content": "hi"}]})
            assert r.status_code == 200 and r.json()["model"] == (name or "base")
    assert [r.adapter for r in sch.requests] == [1, 0, -1, -1, -1]
