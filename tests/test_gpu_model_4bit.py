"""GPU: a model's change to 4-bit weights where it is refused."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

NAMES = ("w_qkv", "w_o", "w_gate_up", "w_down")


def _model(dev, intermediate=672, dtype=torch.bfloat16):
    from minimal_inference_amd.model import Model, ModelConfig

    cfg = ModelConfig(hidden_size=256, num_attention_heads=7, num_key_value_heads=1, head_dim=64, num_hidden_layers=2,
                      intermediate_size=intermediate, vocab_size=4096, max_position_embeddings=512)
    return Model(cfg, dev, dtype=dtype, seed=3, max_positions=512)


@pytest.mark.parametrize("intermediate,dtype", [(688, torch.bfloat16), (672, torch.float16)])
def test_refused_weights_leave_the_model_as_it_was(dev, intermediate, dtype):
    """A width that is no whole number of blocks (of the last projection of a layer), another type."""
    model = _model(dev, intermediate, dtype)
    before = [getattr(L, n) for L in model.layers for n in NAMES]
    with pytest.raises(ValueError):
        model.quantize_weights()
    assert all(a is b for a, b in zip(before, [getattr(L, n) for L in model.layers for n in NAMES]))


def test_quantizing_twice_changes_nothing(dev):
    model = _model(dev)
    model.quantize_weights()
    before = [getattr(L, n) for L in model.layers for n in NAMES]
    model.quantize_weights()
    assert all(a is b for a, b in zip(before, [getattr(L, n) for L in model.layers for n in NAMES]))


def test_refused_under_captured_graphs(dev):
    """A scheduler's graphs hold the addresses of the weights that they were captured with,
    which a change would free: refused while such a scheduler lives, and not after it, nor
    for one without graphs, nor where nothing would change."""
    from minimal_inference_amd.engine import Request, Scheduler

    model = _model(dev)
    plain = Scheduler(model, max_batch_size=2, max_seq_len=64, use_graphs=False)
    sch = Scheduler(model, max_batch_size=2, max_seq_len=64)
    before = [getattr(L, n) for L in model.layers for n in NAMES]
    with pytest.raises(RuntimeError, match="captured"):
        model.quantize_weights()
    assert all(a is b for a, b in zip(before, [getattr(L, n) for L in model.layers for n in NAMES]))
    del sch
    model.quantize_weights()
    sch = Scheduler(model, max_batch_size=2, max_seq_len=64)
    model.quantize_weights()  # (nothing to change)
    tokens = []
    for s in (plain, sch):
        s.submit(Request("a", [1, 2, 3], 5, 0.0))
        request = s.waiting[0]
        s.run()
        tokens.append(request.generated_tokens)
    assert tokens[0] == tokens[1] and len(tokens[0]) == 5
