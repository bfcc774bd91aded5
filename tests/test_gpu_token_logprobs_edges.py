"""Token log probabilities of rows that hold NaN: the alternatives' ids, and
rows whose numbers are fewer than the alternatives asked for."""

import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from qwendopamine_b200 import token_logprobs

pytestmark = pytest.mark.gpu

F32, BF, FH = torch.float32, torch.bfloat16, torch.float16
NAN, NINF = float("nan"), float("-inf")


def ranked(x, k):
    """The k best of each row by falling value, equal ones by rising index, NaN last."""
    x = x.double().cpu().numpy()
    out = []
    for row in x:
        nan = np.isnan(row)
        order = np.lexsort((np.arange(row.size), np.where(nan, 0.0, -row), nan))
        out.append(order[:k])
    return np.stack(out)


# a warp a row; a CTA a row (many rows); a row split over a cluster (few rows)
@pytest.mark.parametrize("rows,V", [(9, 250), (200, 2049), (9, 70001), (9, 151936)])
@pytest.mark.parametrize("dtype", [F32, BF, FH])
@pytest.mark.parametrize("k", [1, 5, 32, 33, 128])
def test_ids_of_rows_with_nan(cuda_device, rows, V, dtype, k):
    gen = torch.Generator().manual_seed(V + k)
    x = (torch.randn(rows, V, generator=gen) * 3).to(dtype)
    x[0] = NAN
    x[1] = NAN  # fewer numbers than alternatives
    x[1, V - k + 1:] = torch.arange(k - 1, 0, -1).to(dtype)
    x[2] = NAN  # as many
    at = torch.randperm(V, generator=gen)[:k]
    x[2, at] = torch.randn(k, generator=gen).to(dtype)
    x[3] = NAN  # one number
    x[3, V // 2] = 1.0
    x[4, ::2] = NAN  # numbers, -inf and NaN
    x[4, 1::2] = NINF
    x[4, 1] = 0.5
    x[5] = NAN  # fewer -inf than alternatives, and nothing else
    x[5, 3:3 + (k + 1) // 2] = NINF
    x[6, V // 3] = NAN
    x[7] = NAN  # neighbours, read by one thread
    x[7, 16:24] = torch.arange(8).to(dtype)
    want = ranked(x, k)
    x = x.to(cuda_device)
    ids = torch.zeros(rows, dtype=torch.int64, device=cuda_device)
    r = token_logprobs(x, ids, top_k=k, entropy=True)
    assert (r.top_ids.cpu().numpy() == want).all()
    assert r.top_logprobs[:8].isnan().all() and r.logprobs[:8].isnan().all()
    assert r.entropy[:8].isnan().all()
    assert r.top_logprobs[8:].isfinite().all()


@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused(cuda_device, grad):
    """No tangent is lost without a word, also where nothing requires a gradient."""
    x = torch.randn(3, 40, device=cuda_device)
    ids = torch.zeros(3, dtype=torch.int64, device=cuda_device)
    plain = token_logprobs(x, ids).logprobs
    with fwAD.dual_level(), torch.set_grad_enabled(grad):
        with pytest.raises(RuntimeError, match="forward"):
            token_logprobs(fwAD.make_dual(x, torch.ones_like(x)), ids)
        assert torch.equal(token_logprobs(x, ids).logprobs, plain)


def test_a_temperature_without_an_inverse_is_refused(cuda_device):
    """Below about 4e-39 log2(e) / temperature is not finite in fp32."""
    x = torch.randn(3, 40, device=cuda_device)
    ids = x.argmax(1)
    for t in (4e-39, 1e-39, 2.0 ** -149):
        with pytest.raises(ValueError, match="temperature"):
            token_logprobs(x, ids, temperature=t)
    r = token_logprobs(x, ids, top_k=2, entropy=True, temperature=1e-38)
    assert not r.logprobs.any() and not r.entropy.any()
    best = x.double().topk(2).values  # the second's is its distance over the temperature
    want = (best[:, 1] - best[:, 0]) / 1e-38
    assert (r.top_ids[:, 0] == ids).all()
    assert ((r.top_logprobs[:, 1] - want).abs() <= 1e-6 * want.abs()).all()


def test_a_vocabulary_beyond_32_bits_is_refused(cuda_device):
    x = torch.zeros(1, 1, device=cuda_device).expand(1, (1 << 32) + 5)
    with pytest.raises(ValueError, match="2.31 - 1 tokens"):
        token_logprobs(x, torch.zeros(1, dtype=torch.int64, device=cuda_device))


def test_capture_in_a_graph(cuda_device):
    for rows, V in ((3, 400), (5, 70001), (300, 5000)):
        x = torch.randn(rows, V, device=cuda_device).to(BF).requires_grad_()
        ids = torch.zeros(rows, dtype=torch.int64, device=cuda_device)
        dl = torch.randn(rows, device=cuda_device)

        def go():
            r = token_logprobs(x, ids, top_k=5, entropy=True)
            return (*r, *torch.autograd.grad((r.logprobs, r.entropy), x, (dl, dl)))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            go()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = go()
        with torch.no_grad():
            x.copy_(torch.randn(rows, V, device=cuda_device))
            ids.copy_(torch.arange(rows))
        graph.replay()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(got, go()))
