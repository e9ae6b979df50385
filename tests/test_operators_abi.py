"""CPU: the C entries of the MXFP4, block-norm and draw operators refuse bad arguments
before any launch, and the oracles agree with hand-made cases."""

from __future__ import annotations

import math

import pytest
import torch

FAKE = 1 << 20  # an aligned address that no refused call reads


def _lib():
    from minimal_inference_amd import _lib

    return _lib, _lib.load()


def test_sizes():
    _, lib = _lib()
    assert lib.mi_mxfp4_codes_size(1, 32) == 1024 and lib.mi_mxfp4_scales_size(1, 32) == 256
    assert lib.mi_mxfp4_codes_size(17, 896) == 2 * 7 * 1024 and lib.mi_mxfp4_scales_size(17, 896) == 2 * 2 * 256
    assert lib.mi_mxfp4_codes_size(0, 32) == 0
    for bad in ((-1, 32), (4, 0), (4, 48), (4, (1 << 20) + 32)):
        assert lib.mi_mxfp4_codes_size(*bad) == 0 and lib.mi_mxfp4_scales_size(*bad) == 0
    assert lib.mi_draw_workspace_size(48, 152064) > lib.mi_draw_workspace_size(1, 152064) > 0
    assert lib.mi_draw_workspace_size(65536, 100) == 0 and lib.mi_draw_workspace_size(1, (1 << 20) + 1) == 0


@pytest.mark.parametrize("change", [
    {"rows": -1}, {"rows": (1 << 22) + 1}, {"n": 0}, {"n": (1 << 24) + 1}, {"k": 48}, {"k": 0}, {"k": (1 << 20) + 32},
    {"x": None}, {"codes": None}, {"scales": None}, {"out": None}, {"x": FAKE + 8}, {"codes": FAKE + 8},
    {"scales": FAKE + 8}, {"out": FAKE + 1}, {"bias": FAKE + 1}, {"x_stride": 56}, {"x_stride": 68},
    {"x_stride": (1 << 22) + 8}, {"out_stride": 31}, {"silu": 1, "bias": FAKE}, {"x_scales": FAKE + 4},
    {"ws": FAKE + 8, "ws_bytes": 1 << 20}])
def test_linear_mxfp4_refuses(change):
    mod, lib = _lib()
    a = dict(x=FAKE, x_stride=64, x_scales=None, codes=FAKE, scales=FAKE, bias=None, out=FAKE, out_stride=32, rows=4,
             n=32, k=64, silu=0, ws=None, ws_bytes=0) | change
    assert lib.mi_linear_mxfp4(*a.values(), None) == mod.MI_ERR_INVALID
    assert mod.last_error().startswith("linear_mxfp4")


def test_mxfp4_matrix_calls_refuse():
    mod, lib = _lib()
    for f in (lib.mi_mxfp4_quantize,):
        for bad in ((None, 64, FAKE, FAKE, 4, 64), (FAKE, 64, None, FAKE, 4, 64), (FAKE, 64, FAKE, None, 4, 64),
                    (FAKE + 2, 64, FAKE, FAKE, 4, 64), (FAKE, 60, FAKE, FAKE, 4, 64), (FAKE, 68, FAKE, FAKE, 4, 64),
                    (FAKE, 64, FAKE, FAKE, -4, 64), (FAKE, 64, FAKE, FAKE, 4, 40)):
            assert f(*bad, None) == mod.MI_ERR_INVALID
    for bad in ((None, FAKE, FAKE, 64, 4, 64), (FAKE, FAKE, FAKE, 32, 4, 64), (FAKE, FAKE, FAKE + 8, 64, 4, 64)):
        assert lib.mi_mxfp4_dequantize(*bad, None) == mod.MI_ERR_INVALID
    for f in (lib.mi_mxfp4_pack, lib.mi_mxfp4_unpack):
        for bad in ((None, FAKE, FAKE, FAKE, 4, 64), (FAKE, FAKE, FAKE + 4, FAKE, 4, 64), (FAKE, FAKE, FAKE, FAKE, 4, 33)):
            assert f(*bad, None) == mod.MI_ERR_INVALID


@pytest.mark.parametrize("change", [
    {"rows": -1}, {"rows": 1 << 31}, {"rows": (1 << 22) + 1}, {"xos": 0}, {"xos": 56}, {"hs": 0}, {"hidden": 12}, {"hidden": 0}, {"hidden": 16392}, {"x": None}, {"y": None},
    {"post": None}, {"weight": None}, {"x_out": None}, {"h_out": None}, {"x": FAKE + 8}, {"ys": 68}, {"hs": 60},
    {"gate": FAKE + 8, "col": 1}, {"gate": FAKE, "gs": 4, "col": 1}, {"gate": FAKE + 1}])
def test_post_norm_refuses(change):
    mod, lib = _lib()
    a = dict(x=FAKE, xs=64, y=FAKE, ys=64, post=FAKE, weight=FAKE, gate=None, gs=0, col=0, x_out=FAKE, xos=64,
             h_out=FAKE, hs=64, rows=4, hidden=64, eps=1e-6, scale=1.0) | change
    assert lib.mi_post_norm_add_rms_norm(*a.values(), None) == mod.MI_ERR_INVALID


def test_draw_refuses():
    mod, lib = _lib()
    base = dict(logits=FAKE, stride=100, batch=2, vocab=100, t=FAKE, k=None, p=None, m=None, u=FAKE, out=FAKE, ws=FAKE,
                bytes=1 << 20)
    for change in ({"batch": -1}, {"batch": 65536}, {"vocab": 0}, {"vocab": (1 << 20) + 1}, {"logits": None}, {"t": None},
                   {"u": None}, {"out": None}, {"stride": 99}):
        assert lib.mi_draw(*(base | change).values(), None) == mod.MI_ERR_INVALID
    for change in ({"ws": None}, {"ws": FAKE + 8}, {"bytes": 100}):
        assert lib.mi_draw(*(base | change).values(), None) == mod.MI_ERR_WORKSPACE


def test_oracle_quantisation_by_hand():
    from oracle import mxfp4 as omx

    x = torch.zeros(1, 32, dtype=torch.bfloat16)
    x[0, :9] = torch.tensor([4.0, 0.25, 0.75, 1.25, -1.75, 2.5, 3.5, 7.9, 5.0])
    codes, scales = omx.quantize(x)
    assert scales.tolist() == [[127]]
    assert omx.values(codes, scales)[0, :9].tolist() == [4.0, 0.0, 1.0, 1.0, -2.0, 2.0, 4.0, 6.0, 4.0]
    x[0, 0] = math.inf
    codes, scales = omx.quantize(x)
    assert scales.tolist() == [[255]] and bool(omx.values(codes, scales).isnan().all())


def test_oracle_draw_by_hand():
    from oracle.draw import draw_row

    l = torch.log(torch.tensor([0.1, 0.4, 0.1, 0.4]))
    # (32-bit logits: the two 0.4 are equal, so index 1 comes first)
    assert [draw_row(l, u, 1.0) for u in (0.0, 0.2, 0.55, 0.7)] == [0, 1, 2, 3]
    assert [draw_row(l, u, 1.0, top_k=1) for u in (0.0, 0.99)] == [1, 1]
    assert [draw_row(l, u, 1.0, top_k=3) for u in (0.0, 0.2, 0.99)] == [0, 1, 3]
    assert [draw_row(l, u, 1.0, top_p=0.6) for u in (0.0, 0.6)] == [1, 3]
    assert [draw_row(l, u, 1.0, min_p=0.5) for u in (0.0, 0.6)] == [1, 3]
    assert draw_row(l, 0.3, 0.0) == 1


def test_workspace_of_the_products():
    """k is shared between workgroups where few blocks would leave the chip idle, and
    nowhere that the few-row kernel runs."""
    _, lib = _lib()
    size = lib.mi_linear_mxfp4_workspace_size
    assert size(77, 3584, 18944, 0, 0) > 0 and size(128, 4096, 14336, 0, 1) > 0
    assert size(77, 3584, 18944, 0, 0) % 16 == 0
    assert size(16, 4096, 14336, 0, 0) == 0 and size(64, 4096, 14336, 0, 1) == 0
    assert size(8192, 10240, 8192, 0, 1) == 0
    for bad in ((-1, 32, 64), (100, 0, 64), (100, 32, 48), ((1 << 22) + 1, 32, 64)):
        assert size(*bad, 0, 0) == 0


def test_server_refuses_other_weight_formats():
    from minimal_inference_amd.server import init_engine

    with pytest.raises(ValueError, match="weight_format"):
        init_engine({"weight_format": "int4"})
