"""Values at which the selective scan's arithmetic is easily lost, against the float64
oracle."""

import numpy as np
import pytest
import torch

from oracle import op_oracle as O
from qwendopamine_b200 import selective_scan

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
