"""Token log probabilities on the GPU against the float64 oracle.

Tolerances.  The inputs are exact in both, sums are fp32: a row's results
carry the rounding of the logits' difference to the maximum (2^-24 of at most
a few tens), of 2^y (2^-22 relative) and of the sums (a few 2^-24), so
absolute errors of logp and entropy stay below 2e-5 for logits of size ten
(relative to max(1, |value|)).  Gradients: fp32 relative L2 2e-5 (y up to a
few tens times 2^-24, and 2^-22); 16-bit ones add one rounding, 2^-9 / 2^-12,
doubled; fp16 gradients are kept above its subnormal range by dlogp ~ 1.
"""

import numpy as np
import pytest
import torch

from oracle import op_oracle as O
from qwendopamine_b200 import token_logprobs

pytestmark = pytest.mark.gpu

F32, BF, FH = torch.float32, torch.bfloat16, torch.float16
VALUE = 2e-5
GRAD = {F32: 2e-5, BF: 2.0 ** -8, FH: 2.0 ** -10}
NINF = float("-inf")


def np64(t):
    return t.detach().double().cpu().numpy()


def near(got, want):
    a = np64(got)
    assert a.shape == want.shape
    fin = np.isfinite(want)
    assert (a[~fin] == want[~fin]).all()
    assert (np.abs(a[fin] - want[fin]) <= VALUE * np.maximum(1, np.abs(want[fin]))).all()


def make(dev, rows, V, dtype, seed=0, scale=3.0):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, V, generator=gen) * scale).to(dev, dtype)
    ids = torch.randint(0, V, (rows,), generator=gen).to(dev)
    dl = torch.randn(rows, generator=gen).to(dev)
    de = torch.randn(rows, generator=gen).to(dev)
    return x, ids, dl, de


def check(x, ids, dl, de, k, temperature=1.0, entropy=True):
    leaf = x.detach().requires_grad_()
    r = token_logprobs(leaf, ids, top_k=k, entropy=entropy, temperature=temperature)
    X, I = np64(x), ids.cpu().numpy()
    logp, ent, table = O.token_logprobs(X, I, temperature)
    near(r.logprobs, logp)
    on = I != -100
    if entropy:
        near(r.entropy, ent)
    else:
        assert r.entropy is None
    if k:
        want = O.top_tokens(X, k)
        assert (r.top_ids.cpu().numpy()[on] == want[on]).all()
        near(r.top_logprobs[torch.from_numpy(on).to(x.device)],
             np.take_along_axis(table, want, 1)[on])
        assert (r.top_ids.cpu().numpy()[~on] == -1).all()
    outs, g = ((r.logprobs, r.entropy), (dl, de)) if entropy else ((r.logprobs,), (dl,))
    dx, = torch.autograd.grad(outs, leaf, g)
    assert dx.dtype == x.dtype and dx.shape == x.shape
    want = O.token_logprobs_bwd(X, I, np64(dl), np64(de) if entropy else None, temperature)
    err = np.linalg.norm(np64(dx) - want) / max(np.linalg.norm(want), 1e-30)
    assert err <= GRAD[x.dtype], err
    with torch.no_grad():
        q = token_logprobs(leaf, ids, top_k=k, entropy=entropy, temperature=temperature)
    for a, b in zip(r, q):
        assert (a is None) == (b is None) and (a is None or torch.equal(a, b))


@pytest.mark.parametrize("dtype", [F32, BF, FH])
@pytest.mark.parametrize("rows,V,k", [(1, 1, 1), (3, 2, 2), (5, 7, 3), (4, 8, 0), (2, 9, 9),
                                      (3, 50, 20), (7, 255, 5), (3, 1000, 20), (2, 2049, 128),
                                      (600, 513, 4), (3, 32003, 20), (1, 70001, 100)])
def test_sizes(cuda_device, rows, V, k, dtype):
    check(*make(cuda_device, rows, V, dtype, seed=V), k)


@pytest.mark.parametrize("temperature,entropy,k", [(0.3, True, 4), (1.7, False, 4), (2.5, True, 0),
                                                   (1.0, False, 0)])
def test_options(cuda_device, temperature, entropy, k):
    check(*make(cuda_device, 9, 3001, BF, seed=1), k, temperature, entropy)


@pytest.mark.parametrize("dtype", [F32, BF, FH])
def test_masks(cuda_device, dtype):
    """-inf columns, the type's lowest value as a mask, rows that a mask leaves
    empty, ignored rows (with NaN in them)."""
    x, ids, dl, de = make(cuda_device, 12, 5003, dtype, seed=2)
    x[:, 4000:] = NINF
    x[0] = NINF
    x[1, :3000] = torch.finfo(dtype).min
    x[2] = torch.finfo(dtype).min  # all equal: uniform
    x[3, 1:] = NINF
    ids[:] = ids % 4000
    ids[3] = 0
    ids[4] = -100
    ids[5] = 4500  # a masked token: log probability -inf
    x[6, :] = NINF
    ids[6] = -100
    check(x, ids, dl, de, 6)
    x[4, 7] = float("nan")
    r = token_logprobs(x.requires_grad_(), ids, entropy=True)
    dx, = torch.autograd.grad(r.logprobs, x, dl)
    assert r.logprobs[4] == 0 and r.entropy[4] == 0 and not dx[4].any()
    assert not dx[0].any()


def test_nan_inf_and_foreign_ids(cuda_device):
    x, ids, dl, de = make(cuda_device, 6, 3000, F32, seed=3)
    clean = token_logprobs(x, ids, top_k=3, entropy=True)
    x[0, 5] = float("nan")
    x[1, 2999] = float("inf")
    ids[2], ids[3] = 3000, -7
    r = token_logprobs(x.requires_grad_(), ids, top_k=3, entropy=True)
    assert r.logprobs[:4].isnan().all() and r.entropy[:2].isnan().all()
    assert r.entropy[2:4].isfinite().all()
    for a, b in zip(clean, r):
        assert torch.equal(a[4:], b[4:])
    dx, = torch.autograd.grad(r.logprobs, x, dl)
    assert dx[0].isnan().all() and dx[1].isnan().all()
    assert not dx[2:4].any()  # no log probability to move
    assert dx[4:].isfinite().all()


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("rows", [2, 700])
def test_ties_go_to_the_lowest_index(cuda_device, rows, dtype):
    V, k = 20011, 40
    gen = torch.Generator().manual_seed(4)
    x = torch.randint(0, 3, (rows, V), generator=gen).to(cuda_device, dtype)
    x[0] = 0.0
    x[0, ::2] = -0.0  # equal to 0
    ids = torch.zeros(rows, dtype=torch.int64, device=cuda_device)
    r = token_logprobs(x, ids, top_k=k)
    assert (r.top_ids.cpu().numpy() == O.top_tokens(np64(x) + 0.0, k)).all()
    assert (r.top_ids[0].cpu() == torch.arange(k)).all()


def test_largest_values_with_one_thread(cuda_device):
    """The best tokens all lie in one thread's share of the row, in rising
    order: more candidates than the list holds."""
    rows, V, k = 300, 151936, 100
    gen = torch.Generator().manual_seed(5)
    x = torch.randn(rows, V, generator=gen)
    idx = torch.arange(V)
    few = (idx // 4) % 256 < 101
    x[:, few] = 5 + idx[few].float() / V
    x = x.to(cuda_device)
    ids = torch.zeros(rows, dtype=torch.int64, device=cuda_device)
    r = token_logprobs(x, ids, top_k=k)
    assert (r.top_ids[:3].cpu().numpy() == O.top_tokens(np64(x[:3]), k)).all()
    rising = torch.arange(V, device=cuda_device).float().expand(2, V) / V
    r = token_logprobs(rising, ids[:2], top_k=k)
    assert (r.top_ids.cpu() == torch.arange(V - 1, V - 1 - k, -1)).all()


def test_shapes_strides_and_types_of_ids(cuda_device):
    x, ids, dl, _ = make(cuda_device, 24, 777, BF, seed=6)
    want = token_logprobs(x, ids, top_k=2, entropy=True)
    r = token_logprobs(x.view(2, 3, 4, 777), ids.view(2, 3, 4).int(), top_k=2, entropy=True)
    assert r.logprobs.shape == (2, 3, 4) and r.top_ids.shape == (2, 3, 4, 2)
    for a, b in zip(want, r):
        assert torch.equal(a.flatten(), b.flatten())
    wide = torch.randn(24, 800, device=cuda_device).to(BF)
    wide[:, 5:782] = x
    for leaf in (wide, wide.t().contiguous().t()):
        leaf = leaf.detach().requires_grad_()
        q = token_logprobs(leaf[:, 5:782], ids, top_k=2, entropy=True)
        assert torch.equal(q.top_ids, want.top_ids)
        assert (q.logprobs - want.logprobs).abs().max() < VALUE * 20
        d, = torch.autograd.grad(q.logprobs, leaf, dl)
        ref = O.token_logprobs_bwd(np64(x), ids.cpu().numpy(), np64(dl))
        assert np.linalg.norm(np64(d)[:, 5:782] - ref) <= GRAD[BF] * np.linalg.norm(ref)
        assert not d[:, :5].any() and not d[:, 782:].any()
    one = token_logprobs(x[0], ids[0])
    assert one.logprobs.shape == ()
    none = token_logprobs(x[:0], ids[:0], top_k=3, entropy=True)
    assert none.logprobs.shape == (0,) and none.top_ids.shape == (0, 3)


def test_offsets_beyond_32_bits(cuda_device):
    """More than 2^31 logits: the last rows are as good as the first."""
    V, rows = 151936, 14200
    x = torch.zeros(rows, V, dtype=BF, device=cuda_device)
    x[-1] = torch.randn(V, device=cuda_device).to(BF)
    ids = torch.full((rows,), V - 1, device=cuda_device)
    leaf = x.requires_grad_()
    r = token_logprobs(leaf, ids, top_k=2)
    logp, _, _ = O.token_logprobs(np64(x[-1:]), [V - 1])
    near(r.logprobs[-1:], logp)
    assert abs(float(r.logprobs[-2]) + np.log(V)) < 1e-4
    d, = torch.autograd.grad(r.logprobs, leaf, torch.ones(rows, device=cuda_device))
    ref = O.token_logprobs_bwd(np64(x[-1:]), [V - 1], [1.0])
    assert np.linalg.norm(np64(d[-1:]) - ref) <= GRAD[BF] * np.linalg.norm(ref)


def test_equal_inputs_give_equal_bits(cuda_device):
    for rows in (3, 40, 900):
        x, ids, dl, de = make(cuda_device, rows, 30011, BF, seed=7)

        def go():
            leaf = x.detach().requires_grad_()
            r = token_logprobs(leaf, ids, top_k=10, entropy=True)
            return (*r, *torch.autograd.grad((r.logprobs, r.entropy), leaf, (dl, de)))

        first = go()
        for _ in range(4):
            assert all(torch.equal(a, b) for a, b in zip(first, go()))


def test_another_stream(cuda_device):
    x, ids, _, _ = make(cuda_device, 64, 9001, BF, seed=8)
    want = token_logprobs(x, ids, top_k=3, entropy=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = token_logprobs(x, ids, top_k=3, entropy=True)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_refusals(cuda_device):
    x, ids, _, _ = make(cuda_device, 4, 300, F32)
    with pytest.raises(RuntimeError, match="CUDA"):
        token_logprobs(x.cpu(), ids.cpu())
    with pytest.raises(ValueError, match="token_ids"):
        token_logprobs(x, ids[:3])
    with pytest.raises(ValueError, match="token_ids"):
        token_logprobs(x, ids.float())
    with pytest.raises(ValueError, match="top_k"):
        token_logprobs(x, ids, top_k=301)
    with pytest.raises(ValueError, match="top_k"):
        token_logprobs(x, ids, top_k=-1)
    with pytest.raises(NotImplementedError, match="128"):
        token_logprobs(x, ids, top_k=129)
    with pytest.raises(TypeError):
        token_logprobs(x.double(), ids)
    for t in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="temperature"):
            token_logprobs(x, ids, temperature=t)
    leaf = x.requires_grad_()
    d, = torch.autograd.grad(token_logprobs(leaf, ids).logprobs.sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(d.sum(), leaf)
