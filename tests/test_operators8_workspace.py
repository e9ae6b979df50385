"""CPU: a workspace that lies over another argument is refused, in the products that hold sums there."""

from __future__ import annotations

import ctypes

import pytest

FAKE = 1 << 32  # an aligned address that no refused call reads


def _lib():
    from minimal_inference_amd import _lib

    return _lib, _lib.load()


# 200 rows of a long k: the workgroups share k.  x at 0, its scales at 2^24, W at 2^25, its scales at 2^30, out at 2^31,
# out's scales at 3 2^30.
LINEAR = dict(x=FAKE, xs=16384, xsc=FAKE + (1 << 24), xss=512, w=FAKE + (1 << 25), ws=16384, wsc=FAKE + (1 << 30), wss=512, bias=None,
              out=FAKE + (1 << 31), os=128, osc=None, oss=0, rows=200, n=128, k=16384, silu=0, work=FAKE + (1 << 33), bytes=1 << 28)


@pytest.mark.parametrize("rows,silu,at", [(rows, silu, at) for rows, silu in ((200, 0), (200, 1), (64, 0))
                                          for at in ("x", "xsc", "w", "wsc", "out", "osc" if silu else "bias")])
def test_linear_refuses_a_workspace_over(at, rows, silu):
    mod, lib = _lib()
    a = LINEAR | {"rows": rows, "silu": silu}
    if rows == 64:
        a |= {"n": 4096, "os": 4096}
    need = lib.mi_linear_mxfp8_workspace_size(a["rows"], a["n"], a["k"], silu)
    assert need > 0
    if at == "bias":
        a["bias"] = FAKE + (1 << 34)
    if at == "osc":
        a |= {"osc": FAKE + (3 << 30), "oss": a["n"] // 32}
    a["work"] = a[at] - need + 16  # (its last bytes)
    assert lib.mi_linear_mxfp8(*a.values(), None) == mod.MI_ERR_INVALID
    assert mod.last_error() == "linear_mxfp8: the workspace overlaps another argument"


ADAPT = dict(y=FAKE, ys=64, x=FAKE + (1 << 20), xs=96, xsc=None, xss=0, a=FAKE + (1 << 21), b=FAKE + (1 << 22), scale=FAKE + (1 << 23),
             slots=3, k=96, rank=24, pieces=(48, 16), n_pieces=2, out=FAKE + (1 << 24), os=64, osc=None, oss=0, plan=FAKE + (1 << 25), rows=4,
             silu=0, work=FAKE + (1 << 26), bytes=1 << 24)


@pytest.mark.parametrize("at", ["y", "x", "xsc", "a", "b", "scale", "plan", "in place"])
def test_adapters_refuse_a_workspace_over(at):
    mod, lib = _lib()
    held = (ctypes.c_int32 * 2)(*ADAPT["pieces"])
    a = ADAPT | {"pieces": ctypes.addressof(held)}
    if at == "xsc":
        a |= {"xsc": FAKE + (1 << 19), "xss": 16}
    need = lib.mi_add_adapters_workspace_size(4, 3, 96, 24, 2, 64, 0)
    assert need > 0
    if at == "in place":
        a["out"] = a["y"]
        at = "y"
    a["work"] = a[at] - need + 16
    assert lib.mi_add_adapters(*a.values(), None) == mod.MI_ERR_INVALID
    # (y is out itself in place)
    assert mod.last_error().startswith("add_adapters: ") and "overlaps another argument" in mod.last_error()


# x at 0 (bf16, or codes), its scales at 2^25, W at 2^26, its scales at 2^30, out at 2^31
LINEAR4 = dict(x=FAKE, xs=16384, xsc=None, w=FAKE + (1 << 26), wsc=FAKE + (1 << 30), bias=None, out=FAKE + (1 << 31), os=128, rows=200,
               n=128, k=16384, silu=0, work=FAKE + (1 << 33), bytes=1 << 28)


@pytest.mark.parametrize("mx,at", [(mx, at) for mx in (0, 1) for at in ("x", "w", "wsc", "out", "bias") + (("xsc",) if mx else ())])
def test_linear_mxfp4_refuses_a_workspace_over(at, mx):
    mod, lib = _lib()
    a = LINEAR4 | ({"xsc": FAKE + (1 << 25)} if mx else {})
    need = lib.mi_linear_mxfp4_workspace_size(a["rows"], a["n"], a["k"], 0, mx)
    assert need > 0
    if at == "bias":
        a["bias"] = FAKE + (1 << 34)
    a["work"] = a[at] - need + 16
    assert lib.mi_linear_mxfp4(*a.values(), None) == mod.MI_ERR_INVALID
    assert mod.last_error() == "linear_mxfp4: the workspace overlaps another argument"
