"""Calls of the selective scan, the token sampling and the gradient norm that are
allowed and rare: offsets beyond 32 bits, rows off every alignment, expanded tensors,
another stream, inference mode, one workspace pool for two captured graphs."""

import numpy as np
import pytest
import torch

from oracle import op_oracle as O
from qwendopamine_b200 import (clip_grad_norm_, grad_norm, sample_tokens, selective_scan,
                               selective_scan_step)

pytestmark = pytest.mark.gpu
BF, FH, F32 = torch.bfloat16, torch.float16, torch.float32


def operands(dev, b, t, d, n, dtype=BF, seed=0):
    gen = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen).to(dev, dtype)
    A = -(0.5 + torch.rand(d, n, generator=gen)).to(dev)
    return [rn(b, t, d), rn(b, t, d), A, rn(b, t, n), rn(b, t, n), torch.randn(d, generator=gen).to(dev),
            rn(b, t, d)]


def both(ops, dy):
    """Results and gradients of a call."""
    ops = [o.detach().requires_grad_() for o in ops]
    y, ht = selective_scan(*ops, dt_softplus=True, output_final_state=True)
    return [y.detach(), ht.detach(), *torch.autograd.grad((y, ht), ops, (dy, torch.ones_like(ht)))]


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_rows_whose_offsets_pass_32_bits(cuda_device):
    """1040 rows, 2^22 values apart, in one buffer of 4.4e9 values; the state pool's
    rows 2^31 values apart."""
    rows, d, n = 1040, 40, 16
    ops = operands(cuda_device, 1, rows, d, n)
    dy = torch.randn(1, rows, d, device=cuda_device).to(BF)
    buf = torch.empty(1, rows, 1 << 22, dtype=BF, device=cuda_device)
    far, at = [], 0
    for o in [*ops, dy]:
        if o.ndim == 3:
            view = buf[:, :, at:at + o.shape[2]]
            view.copy_(o)
            at += o.shape[2] + 8
            far.append(view)
        else:
            far.append(o)
    assert same(both(ops, dy), both(far[:-1], far[-1]))
    del buf, far, view
    big = torch.empty((1 << 31) + d * n + 3, dtype=F32, device=cuda_device)
    pool = big.as_strided((2, d, n), (1 << 31, n, 1))
    pool.copy_(torch.randn(2, d, n, device=cuda_device))
    near, one = pool.clone(), [o[:, 0] if o.ndim == 3 else o for o in operands(cuda_device, 2, 1, d, n)]
    y = [selective_scan_step(*one, dt_softplus=True, state=s) for s in (near, pool)]
    assert torch.equal(*y) and torch.equal(near, pool)


def test_logits_whose_offsets_pass_32_bits(cuda_device):
    buf = torch.empty(3, 1 << 30, dtype=FH, device=cuda_device)
    x = buf[:, 5:5 + 3001]
    x.copy_(torch.randn(3, 3001, device=cuda_device) * 3)
    u = torch.tensor([0.1, 0.5, 0.9], device=cuda_device)
    for o in (dict(), dict(top_k=7), dict(top_p=0.7), dict(temperature=0)):
        assert torch.equal(sample_tokens(x, u, **o), sample_tokens(x.contiguous(), u, **o))


def test_a_vocabulary_beyond_the_histograms_places(cuda_device):
    """2^27 + 1 fp16 logits: wide top-p, and more equal values than any list holds."""
    v = (1 << 27) + 1
    x = torch.zeros(1, v, dtype=FH, device=cuda_device)
    x[0, ::2] = -8.0
    u = torch.tensor([0.25], device=cuda_device)
    odd, even = v // 2, v // 2 + 1
    kept = -(-odd // 2)  # of the equal largest, the first half
    got = sample_tokens(x, u, top_p=float(kept / (odd + even * float(np.exp(-8.0)))))
    # the options and uniform numbers are fp32 or the double given; weights' sums 2^-40
    want = 2 * (kept // 4) + 1
    assert abs(int(got) - want) <= 2 and int(got) % 2 == 1
    assert int(sample_tokens(x, u, top_k=10)) == 2 * 2 + 1  # 0.25 * 10: the third of the first ten
    assert int(sample_tokens(x, u, temperature=0)) == 1


@pytest.mark.parametrize("dtype", [BF, FH, F32])
@pytest.mark.parametrize("off", [0, 1, 2, 4])
def test_rows_off_every_alignment(cuda_device, off, dtype):
    """The widths of the asynchronous copies, and none: equal bits."""
    ops = operands(cuda_device, 2, 90, 24, 16, dtype, seed=1)
    dy = torch.randn(2, 90, 24, device=cuda_device).to(dtype)
    want = both(ops, dy)

    def moved(o):
        if o.ndim != 3:
            return o
        wide = torch.full((*o.shape[:2], o.shape[2] + 16 + off), torch.nan, dtype=o.dtype, device=cuda_device)
        wide[..., off:off + o.shape[2]] = o
        return wide[..., off:off + o.shape[2]]

    assert same(want, both([moved(o) for o in ops], moved(dy)))


def test_expanded_tensors(cuda_device):
    x, dt, A, B, C, D, z = operands(cuda_device, 3, 20, 24, 16, F32, seed=2)
    few = [t[:1].clone().requires_grad_() for t in (dt, B, C)]
    full = [t.detach().expand(3, -1, -1).contiguous().requires_grad_() for t in few]
    grads = []
    for dt_, B_, C_ in ([t.expand(3, -1, -1) for t in few], full):
        y, _ = selective_scan(x, dt_, A, B_, C_, D, z, dt_softplus=True)
        leaves = few if not grads else full
        grads.append(torch.autograd.grad(y.sum(), leaves))  # dy is an expanded 1
    for a, b in zip(*grads):
        assert torch.equal(a, b.sum(0, keepdim=True))


def test_another_stream_and_two_calls_at_once(cuda_device):
    ops = [operands(cuda_device, 2, 700, 40, 16, BF, seed=s) for s in (3, 4)]
    dy = torch.randn(2, 700, 40, device=cuda_device).to(BF)
    x, u = torch.randn(40, 5000, device=cuda_device), torch.rand(40, device=cuda_device)
    grads = [torch.randn(100003, device=cuda_device) for _ in range(3)]
    call = lambda o: [*both(o, dy), sample_tokens(x, u, top_p=0.8), *grad_norm(grads, max_norm=1.0)]
    want = [call(o) for o in ops]
    streams = [torch.cuda.Stream() for _ in ops]
    got = [None, None]
    for _ in range(3):
        for i, s in enumerate(streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got[i] = call(ops[i])
        torch.cuda.synchronize()
        assert all(same(g, w) for g, w in zip(got, want))


def test_inference_mode(cuda_device):
    with torch.inference_mode():
        ops = operands(cuda_device, 2, 9, 24, 16, F32, seed=5)
        y, ht = selective_scan(*ops, dt_softplus=True, output_final_state=True)
        pool = torch.zeros(2, 24, 16, device=cuda_device)
        for t in range(9):
            one = [o[:, t] if o.ndim == 3 else o for o in ops]
            last = selective_scan_step(*one, dt_softplus=True, state=pool)
        # the same nine steps, roundings of 2^-20.5 each
        assert float((pool - ht).norm() / ht.norm()) <= 2e-5 and last.shape == (2, 24)
        assert int(sample_tokens(torch.eye(5, device=cuda_device)[2], torch.tensor(0.5, device=cuda_device),
                                 temperature=0)) == 2
        g = torch.ones(10, device=cuda_device)
        clip_grad_norm_([g], 1.0)
        # 1 / (10^0.5 + 1e-6) within the roundings of the norm and the product
        assert float(g[0]) == pytest.approx(10 ** -0.5, rel=1e-6)


def test_two_graphs_with_one_pool(cuda_device):
    """Chunked scans, whose workspaces the graphs' pool hands to both."""
    ops = [operands(cuda_device, 1, 900, 24, 16, BF, seed=s) for s in (6, 7)]
    x, u = torch.randn(3, 9000, device=cuda_device), torch.rand(3, device=cuda_device)
    g = [torch.randn(5000, device=cuda_device) for _ in range(300)]

    def call(o):
        with torch.no_grad():
            y, ht = selective_scan(*o, dt_softplus=True, output_final_state=True)
        return y, ht, sample_tokens(x, u, top_k=20), *grad_norm(g, max_norm=1.0)

    want = [[t.clone() for t in call(o)] for o in ops]
    graphs, outs, pool = [], [], None
    for o in ops:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            outs.append(call(o))
        pool = graph.pool()
        graphs.append(graph)
    for i in (0, 1, 1, 0):
        graphs[i].replay()
        assert same(outs[i], want[i])


@pytest.mark.parametrize("top_p", [1e-30, 1e-6, 0.999999, 1 - 2.0 ** -24])
def test_extreme_top_p(cuda_device, top_p):
    x = (torch.randn(3, 4099, generator=torch.Generator().manual_seed(8)) * 4).to(cuda_device)
    u = torch.tensor([0.0, 0.37, 1.0], device=cuda_device)
    got = sample_tokens(x, u, top_p=top_p).tolist()
    want = [O.sample_token(r, float(v), 1.0, 0, top_p) for r, v in zip(x.double().cpu().numpy(), u.cpu().numpy())]
    assert got == want


def test_a_gradient_of_more_than_two_to_the_31_values(cuda_device):
    g = torch.zeros((1 << 31) + 9, dtype=BF, device=cuda_device)
    g[-1], g[1 << 31] = 3.0, 4.0
    r = clip_grad_norm_([g], 2.5)
    # 5 within fp32, 2.5 / 5.000001 within 2^-23, the values rounded to bf16 (2^-8)
    assert float(r.norm) == 5.0 and float(r.clip_coef) == pytest.approx(0.5, rel=1e-6)
    assert float(g[-1]) == pytest.approx(1.5, rel=2.0 ** -8) and float(g[1 << 31]) == pytest.approx(2.0, rel=2.0 ** -8)
