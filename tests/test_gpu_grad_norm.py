"""Gradient norm and clipping on the GPU against float64.

Tolerances.  The squares of up to 64 values are summed in fp32 (32 in each of
two chains of up to 16 fused steps, then two sums): every term is rounded at most
18 times, 18 * 2^-24 of the sum of squares; half of that of its root, and one
rounding of the result: 2^-24 (9 + 1).  The coefficient has the same error, one
more rounding, and the scaled values one more product and their own rounding
(half a step).
"""

import math

import numpy as np
import pytest
import torch

from qwendopamine_b200 import AdamW, GradNorm, clip_grad_norm_, grad_norm

pytestmark = pytest.mark.gpu

F32, BF, FH = torch.float32, torch.bfloat16, torch.float16
RTOL = 10 * 2.0 ** -24


def norm64(grads, kind=2.0):
    flat = torch.cat([g.detach().double().flatten() for g in grads])
    return float(flat.abs().max()) if kind == math.inf else float((flat * flat).sum().sqrt())


def make(dev, shapes, dtypes, seed=0, scale=1e-3):
    gen = torch.Generator().manual_seed(seed)
    return [(torch.randn(sh, generator=gen) * scale).to(dev, dt) for sh, dt in zip(shapes, dtypes)]


SHAPES = [(1,), (7,), (8,), (9,), (33, 5), (256,), (1000, 3), (4097,), (129, 513), (2, 0), (70001,)]


@pytest.mark.parametrize("kind", [2.0, math.inf])
@pytest.mark.parametrize("dtype", [F32, BF, FH, None])
def test_norm_of_many_sizes(cuda_device, dtype, kind):
    dtypes = [dtype or (F32, BF, FH)[i % 3] for i in range(len(SHAPES))]
    grads = make(cuda_device, SHAPES, dtypes)
    for lists in (grads, *([g] for g in grads if g.numel())):
        want = norm64(lists, kind)
        r = grad_norm(lists, max_norm=0.3 * want, norm_type=kind)
        assert isinstance(r, GradNorm) and all(x.dtype == F32 and x.shape == () for x in r)
        assert abs(float(r.norm) - want) <= RTOL * want
        coef = 0.3 * want / (want + 1e-6)
        assert abs(float(r.clip_coef) - coef) <= (RTOL + 2.0 ** -24) * coef
        assert float(r.found_inf) == 0
        assert float(grad_norm(lists, norm_type=kind).clip_coef) == 1.0
        assert float(grad_norm(lists, max_norm=2 * want + 1, norm_type=kind).clip_coef) == 1.0


def test_more_tensors_than_a_launch_takes(cuda_device):
    grads = make(cuda_device, [(1 + i % 37,) for i in range(777)], [(F32, BF)[i % 2] for i in range(777)])
    r = grad_norm(grads)
    assert abs(float(r.norm) - norm64(grads)) <= RTOL * norm64(grads)


def test_a_tensor_of_many_chunks(cuda_device):
    """More chunks than partial sums at the least chunk, in the last dtype's odd place."""
    x = torch.randn((80 << 20) + 3, device=cuda_device, dtype=BF)[1:]
    r = grad_norm([x])
    want = norm64([x])
    assert abs(float(r.norm) - want) <= RTOL * want
    assert float(grad_norm(x, norm_type=math.inf).norm) == float(x.abs().max())


@pytest.mark.parametrize("dtype", [F32, BF, FH])
@pytest.mark.parametrize("off", [0, 1, 3, 7])
@pytest.mark.parametrize("n", [1, 5, 8, 63, 2049, 20000])
def test_views_off_a_vectors_alignment(cuda_device, dtype, off, n):
    base = make(cuda_device, [(n + 16,)], [dtype], seed=1)[0]
    before = base.clone()
    x = base[off:off + n]
    want = norm64([x])
    assert abs(float(grad_norm([x]).norm) - want) <= RTOL * want
    r = clip_grad_norm_([x], 0.5 * want)
    coef = min(1.0, 0.5 * want / (want + 1e-6))
    wide = before[off:off + n].double() * coef
    step = torch.finfo(dtype).eps / 2 + RTOL + 2.0 ** -23
    # below the least normal number a step does not shrink further
    least = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    assert ((x.double() - wide).abs() <= step * wide.abs() + least).all()
    assert torch.equal(base[:off], before[:off]) and torch.equal(base[off + n:], before[off + n:])
    assert abs(float(r.norm) - want) <= RTOL * want


@pytest.mark.parametrize("dtype,values", [
    (F32, [1e30, 3e38, 1e-30, 0.0]), (F32, [1e-30, 2e-38, 1e-44]), (BF, [3e38, 1e38, 1.0]),
    (BF, [1e-38, 3e-39]), (FH, [6e-8, 6e-5]), (FH, [65504.0, 60000.0])])
@pytest.mark.parametrize("n", [3, 5000])
def test_values_whose_squares_leave_fp32(cuda_device, dtype, values, n):
    x = torch.zeros(n, dtype=dtype, device=cuda_device)
    x[: len(values)] = torch.tensor(values, dtype=torch.float64).to(cuda_device, dtype)[:n]
    want = norm64([x])
    assert 0 < want < 3.4e38
    got = float(grad_norm([x]).norm)
    # the norm itself may be below the normal numbers
    assert abs(got - want) <= RTOL * want + 2.0 ** -150


def test_norm_that_fp32_cannot_hold(cuda_device):
    x = torch.full((100,), 3e38, device=cuda_device)
    r = grad_norm([x], max_norm=1.0)
    assert float(r.norm) == math.inf and float(r.found_inf) == 1 and float(r.clip_coef) == 1
    assert float(grad_norm([x], max_norm=1.0, norm_type=math.inf).norm) == float(x[0])


@pytest.mark.parametrize("kind", [2.0, math.inf])
@pytest.mark.parametrize("dtype", [F32, BF, FH])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("at", [0, 4000, 9999])
def test_values_that_are_not_finite(cuda_device, dtype, kind, bad, at):
    x = make(cuda_device, [(10000,)], [dtype])[0]
    x[at] = bad
    y = make(cuda_device, [(300,)], [dtype], seed=2)[0]
    kept = [x.clone(), y.clone()]
    for order in ([x, y], [y, x]):
        r = clip_grad_norm_(order, 1e-3, norm_type=kind)
        assert float(r.found_inf) == 1 and float(r.clip_coef) == 1
        assert math.isnan(float(r.norm)) if math.isnan(bad) else float(r.norm) == math.inf
    for a, b in zip((x, y), kept):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_zero_gradients_and_empty_tensors(cuda_device):
    z = [torch.zeros(5000, device=cuda_device), torch.zeros(0, device=cuda_device)]
    for kind in (2.0, math.inf):
        r = clip_grad_norm_(z, 0.0, norm_type=kind)
        assert float(r.norm) == 0 and float(r.found_inf) == 0 and float(r.clip_coef) == 0
        assert float(grad_norm(z[1:], max_norm=1.0, norm_type=kind).norm) == 0


def test_limits_of_zero_and_infinity(cuda_device):
    x = make(cuda_device, [(1000,)], [F32])[0]
    y = x.clone()
    assert float(clip_grad_norm_([x], math.inf).clip_coef) == 1 and torch.equal(x, y)
    assert float(clip_grad_norm_([x], 0).clip_coef) == 0 and not x.any()


def test_equal_inputs_give_equal_bits(cuda_device):
    grads = make(cuda_device, SHAPES, [(F32, BF, FH)[i % 3] for i in range(len(SHAPES))])
    a = [float(grad_norm(grads).norm) for _ in range(5)]
    assert len(set(a)) == 1


def test_strided_and_repeated_tensors(cuda_device):
    x = make(cuda_device, [(40, 60)], [F32])[0]
    for view in (x.t(), x[:, ::2], x[::3], x[0].expand(5, 60)):
        assert abs(float(grad_norm([view]).norm) - norm64([view])) <= RTOL * norm64([view])
    assert abs(float(grad_norm([x, x]).norm) - norm64([x, x])) <= RTOL * norm64([x, x])
    want = x.double() * (1e-2 / (norm64([x]) + 1e-6))
    clip_grad_norm_([x.t()], 1e-2)  # fills its memory: its own order does not matter
    assert ((x.double() - want).abs() <= 16 * 2.0 ** -24 * want.abs()).all()


def test_refusals(cuda_device):
    x = torch.randn(64, device=cuda_device)
    for call in (grad_norm, lambda g, **k: clip_grad_norm_(g, 1.0, **k)):
        with pytest.raises(ValueError):
            call([])
        with pytest.raises(ValueError):
            call([x], norm_type=1.0)
        with pytest.raises(RuntimeError):
            call([x.cpu()])
        with pytest.raises(ValueError):
            call([x, x.cpu()])
        with pytest.raises(TypeError):
            call([x.double()])
        with pytest.raises(RuntimeError):
            call([torch.sparse_coo_tensor([[0]], [1.0], (4,), device=cuda_device)])
    with pytest.raises(ValueError):
        grad_norm([x], max_norm=-1.0)
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError):
            clip_grad_norm_([x], bad)
    for bad in ([x[::2]], [x[:40], x[30:]], [x, x], [x[:1].expand(64)]):
        kept = x.clone()
        with pytest.raises(ValueError):
            clip_grad_norm_(bad, 1e-3)
        assert torch.equal(x, kept)


def test_clipping_counts_as_a_change(cuda_device):
    x = torch.randn(100, device=cuda_device, requires_grad=True)
    y = x * 2
    loss = (y * y).sum()
    with torch.no_grad():
        clip_grad_norm_([y.detach()], 1e-3)
    with pytest.raises(RuntimeError, match="inplace operation"):
        loss.backward()


def test_on_another_stream_and_in_a_graph(cuda_device):
    grads = make(cuda_device, [(5000,), (77,)], [BF, F32])
    want = norm64(grads)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        r = grad_norm(grads, max_norm=1e-2)
    torch.cuda.current_stream().wait_stream(side)
    assert abs(float(r.norm) - want) <= RTOL * want
    graphs = []
    for _ in range(2):  # each captured call has its own workspace and results
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            graphs.append((g, grad_norm(grads, max_norm=1e-2)))
    for g, r in graphs * 2:
        for x in grads:
            x.mul_(2)
        want *= 2
        g.replay()
        assert abs(float(r.norm) - want) <= RTOL * want
        assert abs(float(r.clip_coef) - min(1, 1e-2 / (want + 1e-6))) <= 1e-6


def test_with_the_optimizer(cuda_device):
    """A step with the coefficient as grad_scale is the step on clipped gradients,
    and a gradient that is not finite leaves the parameters as they are."""
    gen = torch.Generator().manual_seed(3)
    init = [torch.randn(s, generator=gen).to(cuda_device) for s in ((65, 33), (128,))]
    grads = [torch.randn(s, generator=gen).to(cuda_device) for s in ((65, 33), (128,))]
    after = []
    for fused in (True, False):
        ps = [torch.nn.Parameter(p.clone()) for p in init]
        opt = AdamW(ps, lr=1e-2)
        for p, g in zip(ps, grads):
            p.grad = g.clone()
        if fused:
            r = grad_norm([p.grad for p in ps], max_norm=0.5)
            opt.step(grad_scale=r.clip_coef, found_inf=r.found_inf)
        else:
            clip_grad_norm_([p.grad for p in ps], 0.5)
            opt.step()
        after.append([p.detach().clone() for p in ps])
    for a, b in zip(*after):
        assert (a - b).abs().max() <= 1e-6  # a step of 1e-2, moments that differ by a rounding
    ps[0].grad[3, 3] = math.nan
    r = grad_norm([p.grad for p in ps], max_norm=0.5)
    kept = [p.detach().clone() for p in ps]
    opt.step(grad_scale=r.clip_coef, found_inf=r.found_inf)
    assert all(torch.equal(p, k) for p, k in zip(ps, kept))
