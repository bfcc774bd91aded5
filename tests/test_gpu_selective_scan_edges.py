"""Values at which the selective scan's arithmetic is easily lost, against the float64
oracle."""

import numpy as np
import pytest
import torch

from oracle import op_oracle as O
from qwendopamine_b200 import selective_scan, selective_scan_step

pytestmark = pytest.mark.gpu
F32, BF, FH = torch.float32, torch.bfloat16, torch.float16
HALF_STEP = {F32: 2.0 ** -24, BF: 2.0 ** -8, FH: 2.0 ** -11}  # of a result's rounding


def np64(t):
    return t.detach().double().cpu().numpy()


@pytest.mark.parametrize("dtype", [F32, BF, FH])
@pytest.mark.parametrize("n", [4, 16, 40])
@pytest.mark.parametrize("pairs", [1, 20])
def test_sums_over_channels_that_cancel(cuda_device, pairs, n, dtype):
    """dB and dC where each channel's neighbour takes back all but a 2^-9th of its
    share: what is left is made of digits that operands of 11 bits do not have.

    Of the shares' sum of magnitudes: 4 rows' states and gradients, all of one sign, are
    within 4 * 2^-20.5 (a decay and two products a row) and the products of operands cut
    into two TF32 values within 2^-18, together below 2^-17; and the result's rounding."""
    gen = torch.Generator().manual_seed(30 + pairs)
    B, T, d = 2, 4, 2 * pairs
    two = lambda t, sign=1: torch.stack([t, sign * t], -1).flatten(-2)
    some = lambda *s: torch.rand(*s, generator=gen) + 0.5
    dt = some(B, T, pairs)
    dt = torch.stack([dt, dt * (1 + 2.0 ** -9 * some(B, T, pairs))], -1).flatten(-2)
    A = -two(some(n, pairs)).t().contiguous()
    x, dy = two(some(B, T, pairs)).to(dtype), two(some(B, T, pairs), -1).to(dtype)
    vec = [some(B, T, n).to(dtype) for _ in range(2)]
    ops = [t.to(cuda_device) for t in (x, dt, A, *vec)]
    leaves = [t.requires_grad_() for t in ops[3:]]
    y, _ = selective_scan(*ops)
    got = torch.autograd.grad(y, leaves, dy.to(cuda_device))
    # each channel its own group: the shares
    wide = [np.repeat(np64(v)[:, :, None], d, 2) for v in vec]
    g = O.selective_bwd(*(np64(t) for t in (x, dt, A)), *wide, None, None, None, False, None, np64(dy))
    for v, k in zip(got, "BC"):
        want, size = g[k].sum(2), np.abs(g[k]).sum(2)
        assert (np.abs(want) < size * 2.0 ** -6).all()
        assert (np.abs(np64(v) - want) <= HALF_STEP[dtype] * np.abs(want) + 2.0 ** -17 * size).all()


@pytest.mark.parametrize("dtype,dtdtype", [(F32, F32), (BF, F32), (BF, BF), (FH, FH)])
@pytest.mark.parametrize("off", [1, 2, 3, 4, 6, 8, 12])
@pytest.mark.parametrize("d,n", [(24, 20), (20, 10)])
def test_groups_in_rows_off_every_alignment(cuda_device, d, n, off, dtype, dtdtype):
    """Two groups of 12 or 10 channels and 20 or 10 states: their first columns are
    aligned otherwise than the rows, and their last pieces are empty.  Equal bits."""
    gen = torch.Generator().manual_seed(32)
    B, T, g = 2, 50, 2
    rn = lambda *s, dtype=dtype: torch.randn(*s, generator=gen).to(cuda_device, dtype)
    A = -(torch.rand(d, n, generator=gen) + 0.5).to(cuda_device)
    ops = [rn(B, T, d), rn(B, T, d, dtype=dtdtype), A, rn(B, T, g, n), rn(B, T, g, n), rn(d, dtype=F32), rn(B, T, d)]
    dy = rn(B, T, d)

    def moved(o):
        if o.ndim < 3:
            return o
        flat = o.flatten(2)
        wide = torch.full((B, T, 64), torch.nan, dtype=o.dtype, device=cuda_device)
        wide[..., off:off + flat.shape[2]] = flat
        return wide[..., off:off + flat.shape[2]].unflatten(2, o.shape[2:])

    def both(ops, dy):
        leaves = [o.detach().requires_grad_() for o in ops]
        y, ht = selective_scan(*leaves, dt_softplus=True, output_final_state=True)
        return [y.detach(), ht.detach(), *torch.autograd.grad((y, ht), leaves, (dy, torch.ones_like(ht)))]

    want, got = both(ops, dy), both([moved(o) for o in ops], moved(dy))
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("dtype", [F32, BF, FH])
@pytest.mark.parametrize("n", [4, 16, 40])
def test_infinity_reaches_the_vectors_gradients(cuda_device, n, dtype):
    """One infinite x or dy: dB and dC are infinite where their sums are, not NaN."""
    gen = torch.Generator().manual_seed(31)
    T, d, at = 70, 12, 30
    rn = lambda *s: torch.randn(*s, generator=gen)
    for name in ("x", "dy"):
        # decays of 0.8 and more: 40 steps keep an infinite state infinite, and finite ones finite
        v = dict(x=rn(1, T, d).to(dtype), dt=(torch.rand(1, T, d, generator=gen) + 0.5).to(dtype),
                 A=-0.1 * torch.rand(d, n, generator=gen), B=rn(1, T, n).to(dtype), C=rn(1, T, n).to(dtype),
                 dy=rn(1, T, d).to(dtype))
        v[name][0, at, 5] = torch.inf
        ops = [v[k].to(cuda_device) for k in ("x", "dt", "A", "B", "C")]
        leaves = [t.requires_grad_() for t in ops[3:]]
        y, _ = selective_scan(*ops)
        got = torch.autograd.grad(y, leaves, v["dy"].to(cuda_device))
        with np.errstate(invalid="ignore"):
            g = O.selective_bwd(*(np64(v[k]) for k in ("x", "dt", "A", "B", "C")), None, None, None, False, None,
                                np64(v["dy"]))
        for u, k in zip(got, "BC"):
            a, want = np64(u), g[k]
            assert np.isinf(want).any() and not np.isnan(want).any()
            assert np.array_equal(np.isinf(a), np.isinf(want)) and not np.isnan(a).any()
            assert np.array_equal(a[np.isinf(want)], want[np.isinf(want)])


def test_every_nan_reaches_the_vectors_gradients(cuda_device):
    """NaN of a gradient whose bits are all in the lower half of the word."""
    gen = torch.Generator().manual_seed(33)
    T, d, n, at = 40, 10, 16, 21
    rn = lambda *s: torch.randn(*s, generator=gen).to(cuda_device)
    ops = [rn(1, T, d), torch.rand(1, T, d, generator=gen).to(cuda_device), -rn(d, n).abs(), rn(1, T, n), rn(1, T, n)]
    leaves = [t.requires_grad_() for t in ops[3:]]
    dy = rn(1, T, d)
    dy.view(torch.int32)[0, at, 3] = 0x7F800001
    y, _ = selective_scan(*ops)
    dB, dC = torch.autograd.grad(y, leaves, dy)
    row = torch.arange(T, device=cuda_device)[None, :, None].expand(1, T, n)
    assert torch.equal(dB.isnan(), row <= at) and torch.equal(dC.isnan(), row == at)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("n", [1, 3, 6, 12, 20, 33])
@pytest.mark.parametrize("skip", [False, True])
def test_infinity_in_states_that_do_not_fill_their_lanes(cuda_device, skip, n, dtype):
    """One infinite x, dt or dy, everything else positive: sums that are infinite are
    not NaN for the states that the lanes hold beyond the last, nor for a D that is not
    there (with a positive one the same sums are infinite)."""
    gen = torch.Generator().manual_seed(34)
    T, d, at = 150, 10, 70
    some = lambda *s: torch.rand(*s, generator=gen) + 0.5
    for name in ("x", "dt", "dy"):
        # decays of 0.97 and more: 150 steps keep what is infinite, and what is not
        v = dict(x=some(1, T, d).to(dtype), dt=some(1, T, d).to(dtype), A=-0.02 * some(d, n), B=some(1, T, n).to(dtype),
                 C=some(1, T, n).to(dtype), h0=some(1, d, n), D=some(d), dy=some(1, T, d).to(dtype))
        v[name][0, at, 5] = torch.inf
        ops = [v[k].to(cuda_device).requires_grad_(name != "dt") for k in ("x", "dt", "A", "B", "C", "h0")]
        y, ht = selective_scan(*ops[:5], v["D"].to(cuda_device) if skip else None, initial_state=ops[5],
                               output_final_state=True)
        args = [*(np64(v[k]) for k in ("x", "dt", "A", "B", "C", "D")), None, None, False, np64(v["h0"])]
        ry, _, rh = O.selective_fwd(*args)
        pairs = [(y, ry), (ht, rh)]
        if name != "dt":
            got = torch.autograd.grad(y, ops, v["dy"].to(cuda_device))
            with np.errstate(invalid="ignore"):
                want = O.selective_bwd(*args, np64(v["dy"]))
            pairs += [(g, want[k]) for g, k in zip(got, ("x", "dt", "A", "B", "C", "h0"))]
        assert any(np.isinf(w).any() for _, w in pairs)
        for a, w in pairs:
            a = np64(a)
            assert np.array_equal(np.isnan(a), np.isnan(w))
            assert np.array_equal(np.isinf(a), np.isinf(w)) and (a[np.isinf(w)] == w[np.isinf(w)]).all()


@pytest.mark.parametrize("n", [1, 3, 16, 20])
def test_infinity_in_a_step(cuda_device, n):
    one = lambda *s: torch.ones(*s, device=cuda_device)
    for k in (0, 1):  # x, dt
        ops = [one(2, 7), one(2, 7), -one(7, n), one(2, n), one(2, n)]
        ops[k][0, 3] = torch.inf
        pool = one(2, 7, n)
        y = selective_scan_step(*ops, state=pool)
        far = torch.zeros(2, 7, dtype=torch.bool, device=cuda_device)
        far[0, 3] = True
        assert torch.equal(y == torch.inf, far) and not y.isnan().any()
        assert torch.equal(pool == torch.inf, far[..., None].expand_as(pool)) and not pool.isnan().any()


def test_softplus_of_all_steps(cuda_device):
    """One token whose y is softplus(dt): the hardware's base-2 exponential is within
    2^-22, its reciprocal within 2^-23, and about four roundings add 2^-22: 3 * 2^-22."""
    v = torch.linspace(-80.0, 20.0, 4096, device=cuda_device)
    one = torch.ones(1, 1, 1, device=cuda_device)
    A = -torch.ones(4096, 1, device=cuda_device)
    y, _ = selective_scan(torch.ones(1, 1, 4096, device=cuda_device), v[None, None], A, one, one, dt_softplus=True)
    x = np64(v)
    want = np.maximum(x, 0) + np.log1p(np.exp(-np.abs(x)))
    assert np.max(np.abs(np64(y)[0, 0] / want - 1)) <= 3 * 2.0 ** -22


def test_softplus_of_no_numbers(cuda_device):
    """Infinite steps and NaN, in a scan and in a step."""
    v = torch.tensor([torch.inf, -torch.inf, torch.nan, -200.0, 3e38, -3e38], device=cuda_device)
    one, A = torch.ones(1, 1, 1, device=cuda_device), -torch.ones(6, 1, device=cuda_device)
    want = torch.tensor([torch.inf, 0.0, torch.nan, 0.0, 3e38, 0.0], device=cuda_device)
    y, _ = selective_scan(torch.ones(1, 1, 6, device=cuda_device), v[None, None], A, one, one, dt_softplus=True)
    y1 = selective_scan_step(torch.ones(1, 6, device=cuda_device), v[None], A, one[0], one[0], dt_softplus=True,
                             state=torch.zeros(1, 6, 1, device=cuda_device))
    for a in (y.flatten(), y1.flatten()):
        assert torch.equal(a.nan_to_num(7.0, torch.inf), want.nan_to_num(7.0, torch.inf))


@pytest.mark.parametrize("n", [3, 16])
def test_infinity_in_a_chunk_stays_infinite_behind_it(cuda_device, n):
    """Decays that are not zero, and whose product over a chunk of the time axis is."""
    gen = torch.Generator().manual_seed(35)
    T, d, at = 400, 10, 200
    some = lambda *s: torch.rand(*s, generator=gen) + 0.5
    for name in ("x", "dy"):
        v = dict(x=some(1, T, d), dt=some(1, T, d), A=-3.0 * some(d, n), B=some(1, T, n), C=some(1, T, n), dy=some(1, T, d))
        v[name][0, at, 5] = torch.inf
        ops = [v[k].to(cuda_device).requires_grad_() for k in ("x", "dt", "A", "B", "C")]
        y, ht = selective_scan(*ops, output_final_state=True)
        dx, = torch.autograd.grad(y, ops[:1], v["dy"].to(cuda_device))
        far = torch.zeros(1, T, d, dtype=torch.bool, device=cuda_device)
        far[0, at:, 5] = name == "x"
        assert torch.equal(y == torch.inf, far) and not y.isnan().any()
        assert torch.equal(ht == torch.inf, far[:, -1, :, None].expand_as(ht)) and not ht.isnan().any()
        far[0, :at + 1, 5] = name == "dy"
        far[0, at + 1:] = False
        if name == "x":
            far[:] = False
        assert torch.equal(dx == torch.inf, far) and not dx.isnan().any()
