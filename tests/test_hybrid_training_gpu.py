"""KDA and attention layers trained together and then served (examples/hybrid_training.py)."""

import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "examples"))

pytestmark = pytest.mark.gpu


def test_the_trained_model_serves_what_it_was_trained_to():
    import hybrid_training
    losses, off = hybrid_training.main()
    assert all(b == b for b in losses) and losses[-1] < 0.9 * losses[0]
    # four bf16 layers in series, one way and the other: the bound of the serving example
    assert off <= 3e-2


def test_every_parameter_of_the_attention_layer_is_trained():
    import hybrid_serving
    import hybrid_training
    torch.manual_seed(1)
    model = hybrid_serving.Hybrid().to("cuda:0")
    x = torch.randn(1, 70, 512, device="cuda:0").bfloat16()
    hybrid_training.forward(model, x).float().square().mean().backward()
    for layer, kind in zip(model.layers, model.pattern):
        if kind != "K":
            for name, p in layer.named_parameters():
                assert p.grad is not None and torch.isfinite(p.grad).all() and bool((p.grad != 0).any()), name
