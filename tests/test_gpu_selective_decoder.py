"""The operators together: a selective layer against its formulas in 64 bits, a
training step that is left out for a gradient that is not finite, prompts and single
tokens against the whole sequence, sampling behind them, and all of it captured.

Tolerances (relative L2, fp32 parameters and inputs).  The layer is five matrix
products of at most 256 terms, each within 256^0.5 * 2^-24 = 2^-20 of its result, and
the scan within 2e-5; gradients pass through twice as many: 4e-5 for the result, 1e-4
for gradients.
"""

import importlib.util
import os

import numpy as np
import pytest
import torch
import torch.nn.functional as F

from oracle import op_oracle as O
from qwendopamine_b200 import AdamW, sample_tokens

pytestmark = pytest.mark.gpu
PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                    "selective_decoder.py")


@pytest.fixture(scope="module")
def ex():
    spec = importlib.util.spec_from_file_location("selective_decoder", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def plain_layer(p, h, rank, states):
    """SelectiveLayer.forward from its parameters, in the parameters' type."""
    x, z = (h @ p["in_proj.weight"].T).chunk(2, -1)
    w = p["conv.weight"]
    x = F.conv1d(F.pad(x.transpose(1, 2), (w.shape[-1] - 1, 0)), w, p["conv.bias"], groups=w.shape[0])
    x = F.silu(x).transpose(1, 2)
    dt, B, C = (x @ p["x_proj.weight"].T).split([rank, states, states], -1)
    dt = F.softplus(dt @ p["dt_proj.weight"].T + p["dt_bias"])
    A = -p["A_log"].exp()
    state, out = torch.zeros(h.shape[0], *A.shape, dtype=h.dtype), []
    for t in range(h.shape[1]):
        state = torch.exp(dt[:, t, :, None] * A) * state + (dt * x)[:, t, :, None] * B[:, t, None]
        out.append((state * C[:, t, None]).sum(-1))
    y = (torch.stack(out, 1) + p["D"] * x) * F.silu(z)
    return y @ p["out_proj.weight"].T


def far(a, b):
    a, b = a.detach().double().cpu(), b.detach().double()
    return float((a - b).norm() / b.norm())


def test_layer_against_its_formulas(ex, cuda_device):
    torch.manual_seed(3)
    layer = ex.SelectiveLayer(64, states=16).to(cuda_device)
    h = torch.randn(2, 37, 64, device=cuda_device, requires_grad=True)
    dy = torch.randn(2, 37, 64, device=cuda_device)
    y = layer(h)
    y.backward(dy)
    p = {k: v.detach().double().cpu().requires_grad_() for k, v in layer.named_parameters()}
    h64 = h.detach().double().cpu().requires_grad_()
    want = plain_layer(p, h64, layer.rank, layer.states)
    want.backward(dy.double().cpu())
    assert far(y, want) <= 4e-5
    assert far(h.grad, h64.grad) <= 1e-4
    for k, v in layer.named_parameters():
        assert far(v.grad, p[k].grad) <= 1e-4, k


def test_a_step_that_is_not_finite_is_left_out(ex, cuda_device):
    torch.manual_seed(4)
    model = ex.Decoder(layers=2).to(cuda_device, torch.bfloat16)
    opt = AdamW(model.parameters(), lr=1e-3)
    ids = torch.randint(0, ex.VOCAB, (4, 40), device=cuda_device)
    _, r = ex.train_step(model, opt, ids)
    assert float(r.found_inf) == 0 and 0 < float(r.norm) < float("inf")
    assert float(r.clip_coef) == pytest.approx(min(1.0, 1.0 / (float(r.norm) + 1e-6)), rel=1e-6)
    got = torch.stack([p.grad.double().square().sum() for p in model.parameters()]).sum().sqrt()
    assert float(r.norm) == pytest.approx(float(got), rel=1e-6)
    hook = model.embed.weight.register_hook(lambda g: g + torch.inf)
    before = [p.detach().clone() for p in model.parameters()]
    _, r = ex.train_step(model, opt, ids)
    hook.remove()
    assert float(r.found_inf) == 1
    assert all(torch.equal(a, b) for a, b in zip(before, model.parameters()))
    ex.train_step(model, opt, ids)
    assert not all(torch.equal(a, b) for a, b in zip(before, model.parameters()))


def test_prompt_and_tokens_follow_the_whole(ex, cuda_device):
    """Layer by layer in fp32: the prompt's states carry the tokens behind it."""
    torch.manual_seed(5)
    layer = ex.SelectiveLayer(64).to(cuda_device)
    h = torch.randn(3, 20, 64, device=cuda_device)
    with torch.no_grad():
        whole = layer(h)
        for cut in (1, 2, 9, 19):
            cache = layer.cache(3)
            slots = torch.arange(3, dtype=torch.int32, device=cuda_device)
            got = [layer.prompt(h[:, :cut], cache)]
            got += [layer.step(h[:, t], cache, slots)[:, None] for t in range(cut, 20)]
            # both are within 4e-5 of the formulas
            assert far(torch.cat(got, 1), whole.double().cpu()) <= 8e-5


def test_example_runs_and_samples_by_the_rules(ex, cuda_device):
    r = ex.main(steps=3)
    assert np.isfinite(r["losses"]).all() and np.isfinite(r["norms"]).all()
    ids = np.array(r["sampled"])
    assert ids.shape == (4, 12) and ids.min() >= 0 and ids.max() < ex.VOCAB


def test_captured_serving_step(ex, cuda_device):
    """One token through the layer and the sampling, captured and replayed."""
    torch.manual_seed(6)
    layer = ex.SelectiveLayer(64).to(cuda_device, torch.bfloat16)
    head = torch.randn(500, 64, device=cuda_device, dtype=torch.bfloat16) * 0.5
    h, u = torch.randn(4, 64, device=cuda_device, dtype=torch.bfloat16), torch.rand(4, device=cuda_device)
    slots = torch.tensor([3, 0, 2, 1], dtype=torch.int32, device=cuda_device)
    cache, logits = layer.cache(4), torch.empty(4, 500, device=cuda_device, dtype=torch.bfloat16)

    def step(cache):
        torch.mm(layer.step(h, cache, slots), head.T, out=logits)
        return sample_tokens(logits, u, temperature=0.8, top_k=40, top_p=0.9)

    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(layer.cache(4))
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ids = step(cache)
        for c in cache:
            c.zero_()
        other = layer.cache(4)
        for i in range(3):
            h.copy_(torch.randn(4, 64, device=cuda_device))
            u.copy_(torch.rand(4, device=cuda_device))
            g.replay()
            got, rows = ids.tolist(), logits.double().cpu().numpy()
            assert got == step(other).tolist()
            assert all(torch.equal(a, b) for a, b in zip(cache, other))
            want = [O.sample_token(x, float(v), 0.8, 40, 0.9) for x, v in zip(rows, u.cpu().numpy())]
            assert got == want
        del g
