"""Rows for which the token sampling's short ways do not suffice, against the float64
oracle."""

import numpy as np
import pytest
import torch

from oracle import op_oracle as O
from qwendopamine_b200 import sample_tokens

pytestmark = pytest.mark.gpu


def near_miss(gap, many):
    """A row of 10 large values, then ``many`` equal ones ``gap`` below, and the top-p
    that 1000 of these make the ten fall short of by a millionth.

    Nine of the ten lie a 4096th of a bin (of 46 to a logit), less a tenth, further down
    than the histogram's whole 4096ths say: their weight is taken for 4.8e-6 more than
    it is, and half of that is what top-p asks beyond it."""
    m = np.float32(6.0)
    x1 = np.float32(m - np.float32((20 + (2048 + 0.9) / 4096) / 46))
    w1, w0 = np.exp(float(x1) - 6.0), np.exp(-float(gap))
    place = np.float32(m - x1) * np.float32(46.0)
    over = (float(place) * 4096 % 1) / 4096 / 46
    assert 4e-6 < over < 5.3e-6
    row = np.full(6000, -np.inf, dtype=np.float32)
    row[3:12], row[20] = x1, m
    row[40:40 + many] = m - np.float32(gap)
    return row, (1 + 9 * w1 * (1 + over / 2)) / (1 + 9 * w1 + 1000 * w0)


def test_top_p_behind_equal_values_at_top_k(cuda_device):
    """3000 equal logits at the top-k bound (more than a list holds: the first 1000 are
    kept), and a top-p whose first window misses: the bound that top-k left stands."""
    row, top_p = near_miss(6.0, 3000)
    u = np.array([0.0, 0.3, 0.9, 0.999, 0.9999, 0.99999, 1 - 2.0 ** -24], dtype=np.float32)
    want = [O.sample_token(row, float(v), 1.0, 1010, top_p) for v in u]
    assert want[-1] == 40 and want[3] < 40  # ten large values and one of the others
    x = torch.from_numpy(np.stack([row] * len(u))).to(cuda_device)
    got = sample_tokens(x, torch.from_numpy(u).to(cuda_device), top_k=1010, top_p=top_p)
    assert got.tolist() == want


@pytest.mark.parametrize("gap,many", [(6.0, 1000), (16.0, 1000), (6.0, 1990)])
def test_a_gap_behind_a_window_that_misses(cuda_device, gap, many):
    row, top_p = near_miss(gap, many)
    u = np.concatenate([[0.0, 0.5, 0.99], 1 - 2.0 ** -np.arange(10, 25.0)]).astype(np.float32)
    want = [O.sample_token(row, float(v), 1.0, 0, top_p) for v in u]
    assert want[-1] >= 40
    x = torch.from_numpy(np.stack([row] * len(u))).to(cuda_device)
    assert sample_tokens(x, torch.from_numpy(u).to(cuda_device), top_p=top_p).tolist() == want


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("options", [dict(), dict(top_p=0.7), dict(top_k=600), dict(min_p=0.5), dict(temperature=0.0)])
def test_zeros_of_both_signs_are_equal(cuda_device, options, dtype):
    """The largest logits are zeros, some of them negative ones."""
    gen = torch.Generator().manual_seed(4)
    x = torch.where(torch.rand(40, 5000, generator=gen) < 0.5, 0.0, -0.0)
    x[20:, ::3] = -1.0
    u = torch.rand(40, generator=gen)
    want = [O.sample_token(r, float(v), **options) for r, v in zip(x.numpy(), u.numpy())]
    got = sample_tokens(x.to(cuda_device, dtype), u.to(cuda_device), **options)
    assert got.tolist() == want
