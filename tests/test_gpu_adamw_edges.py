"""AdamW on the GPU: calls at the edges of what the entry points take."""

import numpy as np
import pytest
import torch

from qwendopamine_b200 import AdamW, adamw_step

pytestmark = pytest.mark.gpu

BF, F8 = torch.bfloat16, torch.float8_e4m3fn


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


@pytest.mark.parametrize("bits", [32, 8])
def test_roots_of_second_moments(cuda_device, bits):
    """Second moments from the smallest fp32 value up, with an eps below their
    roots: the update divides by the root, and the codes hold it.

    With no first-moment and second-moment gradient (g = 0, beta2 = 1/2) v' = v / 2
    is exact above 2^-148, so the change of a parameter is lr m' / (root' + eps):
    one rounding each of a few operations, and 2^-22 of the root and of the
    reciprocal: 2e-6 in all, and the root of v' (subnormal ones exact in fp32)
    enters as it is."""
    e = np.arange(-147, 120).astype(np.float64)
    more = np.random.default_rng(0).uniform(1, 2, (6, e.size))
    v = np.concatenate([m * 2.0 ** e for m in (1.0, 1.9999, *more)]).astype(np.float32)
    # beta2 v with beta2 = 1/2, rounded as fp32 has it
    half = (v * np.float32(0.5)).astype(np.float64)
    want_root = np.sqrt(half)
    n = v.size
    dev = cuda_device
    if bits == 32:
        # m' = m / 2 such that the step is lr * m' / root = about lr
        m = (want_root * 2).astype(np.float32)
        args = [torch.from_numpy(m).to(dev)], [torch.from_numpy(v).to(dev)]
        p = [torch.zeros(n, device=dev)]
        adamw_step(p, [torch.zeros(n, device=dev)], *args, step=400, lr=1e-3, betas=(0.5, 0.5),
                   eps=1e-30, weight_decay=0.0)
        mm = m.astype(np.float64) / 2
        want = -1e-3 * mm / (want_root + 1e-30)
        got = p[0].double().cpu().numpy()
        assert (np.abs(got - want) <= 2e-6 * np.abs(want)).all()
        return
    # 8 bits: a gradient alone in its block, v' = g^2 / 2; its root is the block's
    # largest value, so its scale is root / 448, and the step is lr m' / root
    g = np.zeros((n, 256), dtype=np.float32)
    g[:, 3] = np.sqrt(v.astype(np.float64)).astype(np.float32)
    sq = (g[:, 3] * g[:, 3] * np.float32(0.5)).astype(np.float64)  # rounded step by step
    keep = sq > 0
    want_root = np.sqrt(sq)
    p = torch.zeros(n * 256, device=dev)
    codes = [torch.zeros(n * 256, dtype=torch.uint8, device=dev).view(F8) for _ in range(2)]
    sm, sv = torch.zeros(n, device=dev), torch.zeros(n, device=dev)
    adamw_step([p], [torch.from_numpy(g).to(dev).view(-1)], [codes[0]], [codes[1]], step=400,
               lr=1e-3, betas=(0.5, 0.5), eps=1e-32, weight_decay=0.0, exp_avg_scales=[sm],
               exp_avg_sq_scales=[sv])
    got = sv.double().cpu().numpy() * 448
    # the root's rounding (twice that in rare cases), 1 / 448's and the product's, each
    # at most 2^-24
    assert (np.abs(got - want_root)[keep] <= 5 * 2.0 ** -24 * want_root[keep]).all()
    step = -1e-3 * (g[:, 3].astype(np.float64) / 2) / (want_root + 1e-32)
    got = p.view(n, 256)[:, 3].double().cpu().numpy()
    assert (np.abs(got - step)[keep] <= 2e-6 * np.abs(step)[keep]).all()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("eps", [1e-38, 1e-39, 2.0 ** -149])
def test_an_eps_below_the_normal_range(cuda_device, bits, eps):
    """Parameters without a gradient so far stay where they are: 0 / eps is 0."""
    p = torch.ones(300, device=cuda_device)
    z = lambda n: torch.zeros(n, device=cuda_device)
    st = [z(300), z(300)] if bits == 32 else [
        torch.zeros(300, dtype=torch.uint8, device=cuda_device).view(F8) for _ in range(2)]
    kw = {} if bits == 32 else dict(exp_avg_scales=[z(2)], exp_avg_sq_scales=[z(2)])
    adamw_step([p], [z(300)], [st[0]], [st[1]], step=1, lr=1e-3, eps=eps, weight_decay=0.0, **kw)
    assert p.eq(1).all()


def test_codes_of_the_largest_first_moments(cuda_device):
    """Blocks whose largest value is near fp32's keep their codes: m' = g / 2, held to
    half a step of e4m3, at most 2^-4 of a normal code or 2^-10 of 448 of the rest."""
    g = torch.zeros(4, 256)
    for i, most in enumerate((3e38, 1.7e38, 9e37, 5e37)):
        g[i] = torch.linspace(-1, 1, 256) * most
    p, z8 = torch.zeros(1024, device=cuda_device), []
    for _ in range(2):
        z8.append(torch.zeros(1024, dtype=torch.uint8, device=cuda_device).view(F8))
    ms, vs = torch.zeros(4, device=cuda_device), torch.zeros(4, device=cuda_device)
    adamw_step([p], [g.view(-1).to(cuda_device)], [z8[0]], [z8[1]], step=1, lr=1e-3,
               betas=(0.5, 0.5), exp_avg_scales=[ms], exp_avg_sq_scales=[vs])
    m = (z8[0].double() * ms.double().repeat_interleave(256)).view(4, 256).cpu()
    want = g.double() / 2
    most = want.abs().amax(1, keepdim=True)
    assert ((m - want).abs() <= 1.0001 * torch.maximum(want.abs() / 16, most * 2.0 ** -10 / 448)).all()


def test_a_refused_step_is_not_counted(cuda_device):
    good = torch.nn.Parameter(torch.ones(8, 4, device=cuda_device))
    strided = torch.nn.Parameter(torch.ones(4, 8, device=cuda_device).t())
    half = torch.nn.Parameter(torch.ones(5, device=cuda_device, dtype=BF))
    opt = AdamW([half, good, strided], lr=1e-2)
    for p in (good, strided, half):
        p.grad = torch.ones_like(p)
    for n in range(3):
        with pytest.raises(ValueError, match="contiguous"):
            opt.step()
        # one launch for each type: the first was taken, the refused one was not
        assert opt.state[half]["step"] == n + 1
        assert opt.state[good]["step"] == opt.state[strided]["step"] == 0
    strided.grad = None
    opt.step()
    # the first step's bias correction: 1e-2 whatever the gradient
    assert (good - (1 - 1e-2 * 1e-2) + 1e-2).abs().max() < 1e-6
    assert opt.state[good]["step"] == 1 and opt.state[half]["step"] == 4


def test_a_sparse_gradient_counts_no_step(cuda_device):
    dense = torch.nn.Parameter(torch.ones(4, 2, device=cuda_device))
    table = torch.nn.Parameter(torch.ones(4, 2, device=cuda_device))
    opt = AdamW([dense, table])
    dense.grad = torch.ones_like(dense)
    table.grad = torch.sparse_coo_tensor([[1]], torch.ones(1, 2), (4, 2)).to(cuda_device)
    with pytest.raises(RuntimeError, match="sparse"):
        opt.step()
    assert opt.state[dense]["step"] == 0 and dense.eq(1).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_capture_of_one_step(cuda_device, bits):
    """A captured step replays with the step count and learning rate it was
    captured with, on the gradients that then lie in the buffers."""
    new = lambda: torch.randn(700, generator=torch.Generator().manual_seed(3)).to(cuda_device)
    z = lambda n: torch.zeros(n, device=cuda_device)
    z8 = lambda n: torch.zeros(n, dtype=torch.uint8, device=cuda_device).view(F8)
    scale = torch.full((), 0.5, device=cuda_device)

    def fresh():
        st = [z(700), z(700)] if bits == 32 else [z8(700), z8(700)]
        sc = {} if bits == 32 else dict(exp_avg_scales=[z(3)], exp_avg_sq_scales=[z(3)])
        return new(), z(700), st, sc

    def step(p, g, st, sc):
        adamw_step([p], [g], [st[0]], [st[1]], step=3, lr=1e-2, grad_scale=scale, **sc)

    a, b = fresh(), fresh()
    step(*fresh())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(*a)
    for seed in (1, 2):
        g = torch.randn(700, generator=torch.Generator().manual_seed(seed)).to(cuda_device)
        a[1].copy_(g)
        b[1].copy_(g)
        graph.replay()
        step(*b)
        assert torch.equal(a[0], b[0])
