"""What the operators refuse before they reach a device."""

import pytest
import torch

from qwendopamine_b200 import clip_grad_norm_


def test_clipping_refuses_parameters():
    """It scales what it is given: parameters in their gradients' place would be scaled."""
    layer = torch.nn.Linear(3, 2)
    before = [p.detach().clone() for p in layer.parameters()]
    for given in (layer.parameters(), list(layer.parameters()), layer.weight, [torch.zeros(2), layer.bias]):
        with pytest.raises(TypeError, match="gradients"):
            clip_grad_norm_(given, 1.0)
    assert all(torch.equal(a, b) for a, b in zip(before, layer.parameters()))
