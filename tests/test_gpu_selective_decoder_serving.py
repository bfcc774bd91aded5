"""The example decoder's serving: GDN-2 and selective layers with their caches against
the whole sequence, and every sampled token against the rules on the logits it was
taken from.

Tolerance (relative L2, fp32).  A GDN-2 layer's and a selective layer's prompt and
single tokens are each within 1e-4 of the whole sequence.  Behind it an error passes
through a norm, at most two more layers and the head, whose sums are of sizes like
their inputs': three layers' errors, each grown to three times itself at most, are
below 1e-3."""

import importlib.util
import os

import pytest
import torch

from oracle import op_oracle as O

pytestmark = pytest.mark.gpu
PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                    "selective_decoder.py")


@pytest.fixture(scope="module")
def ex():
    spec = importlib.util.spec_from_file_location("selective_decoder_serving", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("cut", [1, 20, 70])
def test_tokens_behind_a_prompt_follow_the_whole(ex, cuda_device, cut):
    torch.manual_seed(7)
    model = ex.Decoder().to(cuda_device).eval()
    ids = torch.randint(0, ex.VOCAB, (3, 80), device=cuda_device)
    with torch.no_grad():
        whole = model(ids).double()
        caches, slots = model.caches(3), torch.arange(3, dtype=torch.int32, device=cuda_device)
        got = [model.prompt(ids[:, :cut], caches)]
        got += [model.step(ids[:, t], caches, slots) for t in range(cut, 80)]
    for t, logits in enumerate(got, cut - 1):
        for row in range(3):
            far = (logits[row].double() - whole[row, t]).norm() / whole[row, t].norm()
            assert float(far) <= 1e-3, (t, row)


def test_every_sampled_token_follows_the_rules(ex, cuda_device, monkeypatch):
    torch.manual_seed(8)
    model = ex.Decoder().to(cuda_device, torch.bfloat16).eval()
    options = dict(temperature=[0.0, 0.7, 1.0, 1.3, 1.0], top_k=[0, 20, 0, 50, 1], top_p=[1.0, 1.0, 0.6, 0.95, 1.0],
                   min_p=[0.0, 0.0, 0.0, 0.05, 0.0])
    given = {k: torch.tensor(v, device=cuda_device) for k, v in options.items()}
    seen, fed, sample, step = [], [], ex.sample_tokens, model.step

    def sampled(logits, u, **kw):
        ids = sample(logits, u, **kw)
        seen.append((logits.double().cpu().numpy(), u.cpu().numpy(), ids.tolist()))
        return ids

    def stepped(ids, *rest):
        fed.append(ids.tolist())
        return step(ids, *rest)

    monkeypatch.setattr(ex, "sample_tokens", sampled)
    monkeypatch.setattr(model, "step", stepped)
    prompt = torch.randint(0, ex.VOCAB, (5, 9), device=cuda_device)
    ids = ex.serve(model, prompt, 16, torch.rand(16, 5, device=cuda_device), **given)
    assert len(seen) == 16 and fed == [s[2] for s in seen[:-1]]
    assert ids.t().tolist() == [s[2] for s in seen]
    f32 = {k: v.double().cpu().numpy() for k, v in given.items()}
    for logits, u, got in seen:
        for row in range(5):
            rules = [f32[k][row] for k in ("temperature", "top_k", "top_p", "min_p")]
            assert got[row] == O.sample_token(logits[row], float(u[row]), *rules)
        assert got[0] == logits[0].argmax() and got[4] == logits[4].argmax()
