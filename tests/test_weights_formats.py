"""CPU: what a model's formats mean to loading and sizes."""

from __future__ import annotations

import pytest


def _model():
    from minimal_inference_amd.model import Model, ModelConfig

    return Model(ModelConfig(hidden_size=64, num_attention_heads=2, num_key_value_heads=1, head_dim=32, num_hidden_layers=2,
                             intermediate_size=96, vocab_size=64, max_position_embeddings=32), "cpu", max_positions=32)


def test_a_checkpoint_over_quantised_weights_is_refused_by_their_format():
    """A format is told by what a matrix is, not by what its class is called."""
    from minimal_inference_amd.mxfp4 import MXFP4
    from minimal_inference_amd.mxfp8 import MXFP8
    from minimal_inference_amd.weights import load_weights

    class Held(MXFP4):
        __slots__ = ()

    for w, bits in ((MXFP4.__new__(MXFP4), 4), (Held.__new__(Held), 4), (MXFP8(64, 64, "cpu"), 8)):
        model = _model()
        model.layers[1].w_o = w
        with pytest.raises(ValueError, match=f"{bits}-bit weights"):
            load_weights(model, "nowhere")


def test_weight_bytes_count_adapters():
    import torch

    from minimal_inference_amd.adapters import Adapters

    model = _model()
    before = model.weight_bytes()
    ad = Adapters.__new__(Adapters)  # (made on a GPU alone)
    ad.a, ad.b, ad.scale = torch.zeros(3, 8, 64, dtype=torch.bfloat16), torch.zeros(3, 64, 8, dtype=torch.bfloat16), torch.zeros(3)
    assert ad.nbytes == 2 * 3 * 8 * 128 + 12
    model.layers[1].adapters = {"w_o": ad, "w_down": ad}
    assert model.weight_bytes() == before + 2 * ad.nbytes
