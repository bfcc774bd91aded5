"""AdamW on the GPU: calls at the edges of what the entry points take."""

import pytest
import torch

from qwendopamine_b200 import AdamW, adamw_step

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("master", [False, True])
def test_step_marks_what_it_writes_as_changed(cuda_device, bits, master):
    """A graph that saved a parameter or a state cannot be differentiated after a
    step on it."""
    p = torch.nn.Parameter(torch.randn(300, device=cuda_device).to(BF))
    opt = AdamW([p], state_bits=bits, master_weights=master)
    (p.float() ** 2).sum().backward()
    opt.step()
    held = [p] + [t for t in opt.state[p].values() if isinstance(t, torch.Tensor)]
    versions = [t._version for t in held]
    loss = (p.float() * p.detach()).sum() + (p * p).sum()
    opt.step()
    assert all(t._version > v for t, v in zip(held, versions))
    with pytest.raises(RuntimeError, match="inplace operation"):
        loss.backward()


def test_step_on_tensors_without_a_version(cuda_device):
    with torch.inference_mode():
        p, g, m, v = (torch.full((40,), x, device=cuda_device) for x in (1.0, 1.0, 0.0, 0.0))
        adamw_step([p], [g], [m], [v], step=1, lr=0.5, weight_decay=0.0)
        assert (p - 0.5).abs().max() < 1e-6
