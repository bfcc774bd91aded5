"""The selective scan's and the sampling oracle tied to their definitions (CPU):
gradients to central differences, tokens to the distribution that they stand for."""

import numpy as np
import pytest

from oracle import op_oracle as O

EPS = 1e-6
# central differences in fp64: truncation eps^2 times third derivatives of order
# 10 to 1000, and cancellation 2^-53 * |loss| / eps, about 1e-8
TOL = 1e-6


def differences(f, x):
    g = np.zeros_like(x)
    for i in np.ndindex(*x.shape):
        keep = x[i]
        x[i] = keep + EPS
        hi = f()
        x[i] = keep - EPS
        lo = f()
        x[i] = keep
        g[i] = (hi - lo) / (2 * EPS)
    return g


@pytest.mark.parametrize("cu,groups,gate,plus", [(None, None, True, True), (None, 2, False, False),
                                                 ([0, 3, 3, 4, 7], None, True, True), ([0, 7], 2, True, False)])
def test_selective_gradients_are_the_differences(cu, groups, gate, plus):
    rng = np.random.default_rng(5)
    b, t, d, n = (2, 4, 4, 3) if cu is None else (1, 7, 4, 3)
    s = b if cu is None else len(cu) - 1
    vec = (b, t, n) if groups is None else (b, t, groups, n)
    v = dict(x=rng.standard_normal((b, t, d)), dt=rng.random((b, t, d)), A=-rng.random((d, n)) - 0.2,
             B=rng.standard_normal(vec), C=rng.standard_normal(vec), D=rng.standard_normal(d),
             z=rng.standard_normal((b, t, d)) if gate else None, dt_bias=rng.standard_normal(d) * 0.1,
             h0=rng.standard_normal((s, d, n)))
    dy, dht = rng.standard_normal((b, t, d)), rng.standard_normal((s, d, n))
    args = lambda: (v["x"], v["dt"], v["A"], v["B"], v["C"], v["D"], v["z"], v["dt_bias"], plus, v["h0"])

    def loss():
        y, _, ht = O.selective_fwd(*args(), cu)
        return (y * dy).sum() + (ht * dht).sum()

    g = O.selective_bwd(*args(), dy, dht, cu)
    for k, x in v.items():
        if x is not None:
            assert np.abs(differences(loss, x) - g[k]).max() < TOL, k


def test_sampled_tokens_have_their_probabilities():
    x = np.array([0.0, 2.0, 1.0, 2.0, -np.inf, 1.5])
    u = (np.arange(4000) + 0.5) / 4000

    def share(**options):
        ids = [O.sample_token(x, v, **options) for v in u]
        return np.bincount(ids, minlength=6) / u.size

    p = np.exp(x - 2.0)
    assert np.abs(share() - p / p.sum()).max() < 1e-3
    keep = np.array([0, 1, 0, 1, 0, 0])
    assert np.abs(share(top_k=2) - 0.5 * keep).max() < 1e-3
    assert share(top_k=1)[1] == 1 and share(temperature=0)[1] == 1 and share(top_p=0.1)[1] == 1
    q = p ** 2 * np.array([0, 1, 0, 1, 0, 1])
    assert np.abs(share(temperature=0.5, min_p=0.3) - q / q.sum()).max() < 1e-3
    assert np.abs(share(top_p=0.55) - 0.5 * keep).max() < 1e-3  # the two best reach 0.59
    assert O.sample_token(x, 1.0) == 5 and O.sample_token(x * np.nan, 0.5) == -1
