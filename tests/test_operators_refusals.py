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


FAKE = 1 << 30  # an aligned address that no refused call reads


def _lib():
    from minimal_inference_amd import _lib

    return _lib, _lib.load()


@pytest.mark.parametrize("change", [
    {"out": 0}, {"out": 2}, {"out": -2 * 64 * 3 - 62}, {"out": 2 * 64 * 4 - 2}, {"out_stride": 96, "out": 96 * 2 + 32},
    {"x_stride": 96, "out_stride": 96, "out": 2 * 63}, {"x_stride": 96, "out_stride": 96, "out": -2 * 63},
    {"x_stride": 96, "out_stride": 96, "out": -3 * 96 * 2 - 2}, {"n": 64, "out_stride": 64, "out": 0}, {"rows": 1, "out": 126},
    {"codes": 1 << 20}, {"codes": (1 << 20) - 2048 + 16}, {"codes": (1 << 20) + 448 - 16},
    {"scales": (1 << 20) - 512 + 16}, {"bias": (1 << 20) + 66}, {"bias": (1 << 20) - 62}, {"silu": 1, "codes": (1 << 20) - 4096 + 16},
    {"x_scales": (1 << 20) - 240}, {"x_scales": 1 << 24, "x": (1 << 20) - 1008},
    {"rows": 1 << 22, "x_stride": 128, "out_stride": 136, "out": 136}])
def test_linear_mxfp4_refuses_an_out_over_its_inputs(change):
    """Rows of out that share a byte with x, either of the weight's parts or the bias; the
    weight's rows past its last are part of its tile."""
    mod, lib = _lib()
    a = dict(x=0, x_stride=64, x_scales=None, codes=1 << 28, scales=1 << 29, bias=None, out=1 << 20, out_stride=64, rows=4,
             n=32, k=64, silu=0, ws=None, ws_bytes=0) | change
    for name in ("x", "x_scales", "codes", "scales", "bias", "out"):
        a[name] = None if a[name] is None else a[name] + FAKE
    assert lib.mi_linear_mxfp4(*a.values(), None) == mod.MI_ERR_INVALID
    assert "overlaps" in mod.last_error()


@pytest.mark.parametrize("change", [
    {"h_out": 1 << 24}, {"h_out": (1 << 24) + 3 * 128 + 112}, {"x_out": 16}, {"x_out": -16}, {"x_out": 128}, {"h_out": 16},
    {"x_out": 1 << 20, "xos": 72}, {"h_out": (1 << 20) - 3 * 128}, {"h_out": (1 << 28) + 112}, {"x_out": (1 << 27) - 496},
    {"gate": (1 << 24) + 64, "gs": 0, "col": 1}, {"gate": (1 << 24) + 64, "gs": 72, "col": 1}, {"gate": (1 << 24) + 64, "gs": 0},
    {"gate": (1 << 25) + 128 + 2, "gs": 1}, {"xs": 0, "x_out": 0}, {"xs": 128, "x_out": 0}, {"rows": 1, "h_out": (1 << 24) + 16},
    {"rows": 1, "x_out": 1 << 27}, {"rows": 1 << 22, "h_out": 128}])
def test_post_norm_refuses_outputs_over_other_rows(change):
    """x at 0, y at 2^20, x_out at 2^24, h_out at 2^25, post at 2^27, weight at 2^28: rows of 64
    values, 4 of them."""
    mod, lib = _lib()
    a = dict(x=0, xs=64, y=1 << 20, ys=64, post=1 << 27, weight=1 << 28, gate=None, gs=0, col=0, x_out=1 << 24, xos=64,
             h_out=1 << 25, hs=64, rows=4, hidden=64, eps=1e-6, scale=1.0) | change
    for name in ("x", "y", "post", "weight", "gate", "x_out", "h_out"):
        a[name] = None if a[name] is None else a[name] + FAKE
    assert lib.mi_post_norm_add_rms_norm(*a.values(), None) == mod.MI_ERR_INVALID
    assert "overlaps" in mod.last_error()


def test_a_checkpoint_is_not_loaded_into_4_bit_weights(tmp_path):
    """Refused before a tensor of the model changes."""
    from safetensors.torch import save_file

    from minimal_inference_amd.model import Model, ModelConfig
    from minimal_inference_amd.mxfp4 import MXFP4
    from minimal_inference_amd.weights import load_weights

    cfg = ModelConfig(hidden_size=64, num_attention_heads=2, num_key_value_heads=1, head_dim=32, num_hidden_layers=1,
                      intermediate_size=96, vocab_size=100, max_position_embeddings=64)
    model = Model(cfg, "cpu", max_positions=64)
    save_file({"model.embed_tokens.weight": torch.ones(100, 64, dtype=torch.bfloat16),
               "model.layers.0.mlp.down_proj.weight": torch.ones(64, 96, dtype=torch.bfloat16)},
              str(tmp_path / "model.safetensors"))
    model.layers[0].w_down = MXFP4(64, 96, "cpu")
    before = model.embed.clone()
    with pytest.raises(ValueError, match="4-bit"):
        load_weights(model, str(tmp_path))
    assert torch.equal(model.embed, before)
