"""Token sampling on the GPU against the float64 oracle: the same token in every
row.  Both sides hold weights and sums in fp64 (2e-13 and 1e-16 relative), so a
uniform number would have to fall within 1e-12 of a token's edge for them to
differ; the inputs are fixed by their seeds."""

import math

import numpy as np
import pytest
import torch

from oracle import op_oracle as O
from qwendopamine_b200 import sample_tokens, token_logprobs

pytestmark = pytest.mark.gpu

F32, BF, FH = torch.float32, torch.bfloat16, torch.float16


def want(logits, uniform, **options):
    x, u = logits.double().cpu().numpy(), uniform.double().cpu().numpy()
    pick = lambda o, r: o.double().cpu().numpy()[r] if isinstance(o, torch.Tensor) else o
    return [O.sample_token(x[r], u[r], **{k: pick(o, r) for k, o in options.items()})
            for r in range(x.shape[0])]


def check(logits, uniform, **options):
    got = sample_tokens(logits, uniform, **options)
    assert got.dtype == torch.int64 and got.shape == uniform.shape
    assert got.tolist() == want(logits, uniform, **options)
    return got


def rows(dev, n, V, dtype, seed=0, scale=2.5, lift=8.0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(n, V, generator=gen) * scale
    x[torch.arange(n), torch.randint(0, V, (n,), generator=gen)] += lift
    return x.to(dev, dtype), torch.rand(n, generator=gen).to(dev)


OPTIONS = [dict(), dict(temperature=0.7), dict(top_k=50), dict(top_p=0.9), dict(min_p=0.05),
           dict(temperature=1.3, top_k=20, top_p=0.8, min_p=0.01), dict(top_k=5, top_p=0.3),
           dict(top_p=0.999, min_p=1e-4), dict(top_k=1), dict(temperature=0), dict(top_p=0.0),
           dict(min_p=1.0), dict(top_k=3000, top_p=0.97), dict(temperature=50.0, top_k=40),
           dict(temperature=50.0, top_p=0.5), dict(temperature=0.02, top_p=0.9)]


@pytest.mark.parametrize("options", OPTIONS)
@pytest.mark.parametrize("dtype", [F32, BF, FH])
@pytest.mark.parametrize("n,V", [(1, 1), (3, 2), (5, 9), (40, 1000), (7, 32003)])
def test_options(cuda_device, n, V, dtype, options):
    x, u = rows(cuda_device, n, V, dtype, seed=V)
    check(x, u, **options)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_a_large_vocabulary_split_and_not(cuda_device, dtype):
    x, u = rows(cuda_device, 6, 151936, dtype, seed=1)
    for options in (dict(), dict(top_k=50, top_p=0.9), dict(top_p=0.95), dict(top_k=5000), dict(top_p=0.9999)):
        few = check(x, u, **options)
        # with many rows a row has one CTA, with few eight: the same tokens
        many = sample_tokens(x.repeat(64, 1), u.repeat(64), **options)
        assert torch.equal(many, few.repeat(64))


def test_options_of_each_row(cuda_device):
    x, u = rows(cuda_device, 64, 5000, BF, seed=2)
    gen = torch.Generator().manual_seed(3)
    r = lambda lo, hi: (lo + (hi - lo) * torch.rand(64, generator=gen)).to(cuda_device)
    t, p, q = r(0.0, 2.0), r(0.1, 1.2), r(-0.05, 0.2)
    t[5], t[6], p[7], q[8] = 0.0, -1.0, -0.5, 3.0
    k = torch.randint(-1, 60, (64,), generator=gen).to(cuda_device)
    k[0], k[1] = 5000, 1 << 40
    check(x, u, temperature=t, top_k=k, top_p=p, min_p=q)
    check(x, u, top_k=k.to(torch.int32), temperature=0.8)
    check(x, u, top_p=p.to(BF))


@pytest.mark.parametrize("options", [dict(), dict(top_k=7), dict(top_k=4000), dict(top_p=0.6),
                                     dict(top_k=4500, top_p=0.7), dict(min_p=0.5, top_p=0.4)])
@pytest.mark.parametrize("kind", ["equal", "two", "close", "narrow", "wide", "few"])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_values_that_crowd_a_bin(cuda_device, dtype, kind, options):
    """More equal or close values than a list holds, on either side of the bound."""
    n, V = 4, 9001
    gen = torch.Generator().manual_seed(4)
    z = torch.randn(n, V, generator=gen)
    x = {"equal": z * 0 + 3.0, "two": torch.where(z > 0.2, 1.0, 0.5), "close": 5 + z.round() * 2.0 ** -6,
         "narrow": z * 1e-3, "wide": z * 1e4, "few": (z * 2).round()}[kind].to(cuda_device, dtype)
    u = torch.rand(n, generator=gen).to(cuda_device)
    check(x, u, **options)


def test_equal_logits_rank_by_index(cuda_device):
    x = torch.zeros(5, 151936, device=cuda_device, dtype=BF)
    u = torch.tensor([0.0, 0.25, 0.5, 0.75, 0.999], device=cuda_device)
    assert sample_tokens(x, u, top_k=8000).tolist() == [int(8000 * float(v)) for v in u]
    assert sample_tokens(x, u).tolist() == [int(151936 * float(v)) for v in u]
    assert sample_tokens(x, u, temperature=0).tolist() == [0] * 5


@pytest.mark.parametrize("options", [dict(), dict(top_k=3), dict(top_p=0.8), dict(min_p=0.1)])
@pytest.mark.parametrize("dtype", [F32, BF, FH])
def test_masks(cuda_device, dtype, options):
    x, u = rows(cuda_device, 6, 3001, dtype, seed=5)
    x[:, 1500:] = -math.inf
    x[1, :1499] = -math.inf            # one value left
    x[2] = -math.inf                   # none
    x[3, 700:1400] = torch.finfo(dtype).min
    x[4, ::2] = -math.inf
    got = check(x, u, **options)
    assert got[1] == 1499 and got[2] == -1
    x[0, 5] = math.nan
    x[3, 9] = math.inf
    got = check(x, u, **options)
    assert got[0] == -1 and got[3] == -1
    assert sample_tokens(x, u, temperature=0).tolist() == want(x, u, temperature=0)


def test_ends_of_the_uniform_range(cuda_device):
    x, _ = rows(cuda_device, 4, 1000, F32, seed=6)
    x[:, :10] = -math.inf
    x[:, -10:] = -math.inf
    u = torch.tensor([-3.0, 0.0, 1.0, 7.0], device=cuda_device)
    assert sample_tokens(x, u).tolist() == [10, 10, 989, 989]
    check(x, u, top_k=20)
    u[2] = math.nan
    assert sample_tokens(x, u).tolist() == [10, 10, -1, 989]
    t = torch.tensor([1.0, math.nan, 1.0, 1.0], device=cuda_device)
    assert sample_tokens(x, u, temperature=t).tolist() == [10, -1, -1, 989]
    assert sample_tokens(x, u, top_p=t).tolist() == [10, -1, -1, 989]
    assert sample_tokens(x, u, min_p=t)[1] == -1
    assert sample_tokens(x, u, temperature=1e-300).tolist()[:2] == [int(v) for v in x.argmax(1)[:2]]
    assert sample_tokens(x, u, temperature=1e300).tolist()[:2] == [10, 10]


def test_shapes_strides_and_offsets(cuda_device):
    x, u = rows(cuda_device, 12, 777, BF, seed=7)
    flat = want(x, u, top_p=0.9)
    assert sample_tokens(x.view(3, 4, 777), u.view(3, 4), top_p=0.9).flatten().tolist() == flat
    assert sample_tokens(x[0], u[0], top_p=0.9).tolist() == flat[0]
    wide = torch.full((12, 800), math.inf, device=cuda_device, dtype=BF)
    for off in (0, 1, 5, 8):
        wide[:, off:off + 777] = x
        assert sample_tokens(wide[:, off:off + 777], u, top_p=0.9).tolist() == flat
        wide.fill_(math.inf)
    assert sample_tokens(x.t().contiguous().t(), u, top_p=0.9).tolist() == flat
    assert sample_tokens(x[::2], u[::2], top_p=0.9).tolist() == flat[::2]
    assert sample_tokens(x[:0], u[:0]).shape == (0,)


def test_the_tokens_follow_the_probabilities(cuda_device):
    """An even grid of uniform numbers takes each token as often as it is probable."""
    x = torch.tensor([[0.0, 1.0, 2.0, -1.0, 3.0]], device=cuda_device)
    n = 20000
    u = (torch.arange(n, device=cuda_device) + 0.5) / n
    got = torch.bincount(sample_tokens(x.expand(n, 5), u, temperature=1.5), minlength=5)
    p = torch.softmax(x[0].double() / 1.5, 0)
    assert (got.double() / n - p).abs().max() <= 1.0 / n


def test_refusals(cuda_device):
    x, u = rows(cuda_device, 3, 10, F32)
    for bad in (dict(temperature=-1.0), dict(temperature=math.nan), dict(temperature=math.inf),
                dict(top_k=-1), dict(top_p=1.5), dict(top_p=-0.1), dict(min_p=2.0), dict(min_p=math.nan),
                dict(top_k=torch.ones(2, dtype=torch.int32, device=cuda_device)),
                dict(top_k=torch.ones(3, device=cuda_device)),
                dict(temperature=torch.ones(3, dtype=torch.int64, device=cuda_device))):
        with pytest.raises(ValueError):
            sample_tokens(x, u, **bad)
    for bad in (u[:2], u.double(), u.cpu()):
        with pytest.raises(ValueError):
            sample_tokens(x, bad)
    with pytest.raises(RuntimeError):
        sample_tokens(x.cpu(), u.cpu())
    with pytest.raises(TypeError):
        sample_tokens(x.double(), u)
    with pytest.raises(ValueError):
        sample_tokens(x[:, :0], u)


def test_on_another_stream_and_in_a_graph(cuda_device):
    x, u = rows(cuda_device, 8, 20000, BF, seed=8)
    options = dict(top_k=30, top_p=0.9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = sample_tokens(x, u, **options)
    torch.cuda.current_stream().wait_stream(side)
    assert got.tolist() == want(x, u, **options)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = sample_tokens(x, u, **options)
    for seed in (9, 10):
        x2, u2 = rows(cuda_device, 8, 20000, BF, seed=seed)
        x.copy_(x2)
        u.copy_(u2)
        g.replay()
        assert got.tolist() == want(x, u, **options)


def test_with_the_log_probabilities(cuda_device):
    """What a serving step does: choose, then report the choice."""
    x, u = rows(cuda_device, 16, 4000, BF, seed=11)
    ids = sample_tokens(x, u, temperature=0.7, top_k=5)
    r = token_logprobs(x, ids, temperature=0.7, top_k=5)
    assert (r.top_ids == ids[:, None]).any(1).all()
    assert torch.equal(sample_tokens(x, u, temperature=0), token_logprobs(x, ids, top_k=1).top_ids[:, 0])
