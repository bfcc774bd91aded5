"""What the operators refuse before they reach a device."""

import pytest
import torch

from qwendopamine_b200 import _native as N
from qwendopamine_b200 import clip_grad_norm_


def test_clipping_refuses_parameters():
    """It scales what it is given: parameters in their gradients' place would be scaled."""
    layer = torch.nn.Linear(3, 2)
    before = [p.detach().clone() for p in layer.parameters()]
    for given in (layer.parameters(), list(layer.parameters()), layer.weight, [torch.zeros(2), layer.bias]):
        with pytest.raises(TypeError, match="gradients"):
            clip_grad_norm_(given, 1.0)
    assert all(torch.equal(a, b) for a, b in zip(before, layer.parameters()))


@pytest.mark.parametrize("n,tile", [(1, 64), (8, 64), (9, 32), (16, 32), (17, 16), (32, 16), (33, 8), (64, 8)])
@pytest.mark.parametrize("d,groups", [(4096, 1), (4096, 4), (770, 2), (40, 40)])
def test_memory_of_the_selective_scans_gradient(n, tile, d, groups):
    """What is documented: a state every 16 tokens, and 8 N bytes of scratch a token for
    every tile of channels, of which each group has its own; with it come a state and a
    few sums of each channel for each of up to 592 chunks."""
    t = 8192
    p = N.SelectiveProblem(1, d, groups, n, t, 1, 1, 0, 1, None, d, d, d, groups * n, groups * n, d)
    states = d * (-(-n // 4) * 4) * 4
    lib = N.load()
    assert lib.gdn2_selective_saved_bytes(p) == t // 16 * states
    tiles = groups * -(-(d // groups) // tile)
    more = lib.gdn2_selective_workspace_bytes(p, 1) - tiles * 8 * n * t
    chunks = min(t // 64, -(-592 // tiles))  # of 64 tokens at least, about 592 CTAs
    assert 0 <= more <= chunks * 2 * (states + 8 * d) + 5 * 256
