"""The operators' float64 oracle: its gradients against central differences of
its own forward (no GPU)."""

import numpy as np
import pytest

from oracle import op_oracle as O

STEP = 1e-5
# central differences in float64: truncation ~ STEP^2 = 1e-10, rounding ~
# 1e-16 * |loss| / STEP ~ 1e-10 for losses of order ten
TOL = 1e-7


def differences(f, x):
    out = np.zeros_like(x)
    for i in np.ndindex(x.shape):
        keep = x[i]
        x[i] = keep + STEP
        up = f()
        x[i] = keep - STEP
        down = f()
        x[i] = keep
        out[i] = (up - down) / (2 * STEP)
    return out


@pytest.mark.parametrize("gate", [True, False])
@pytest.mark.parametrize("cu", [None, [0, 0, 1, 4, 4, 7]])
def test_scan_gradients_are_the_differences(gate, cu):
    rng = np.random.default_rng(3)
    B, T, D = (2, 5, 3) if cu is None else (1, 7, 3)
    n = B if cu is None else len(cu) - 1
    v, g = rng.standard_normal((B, T, D)), -rng.random((B, T, D))
    w = rng.random((B, T, D)) if gate else None
    h0, dht = rng.standard_normal((n, D)), rng.standard_normal((n, D))
    dy = rng.standard_normal((B, T, D))

    def loss():
        y, ht = O.scan_fwd(v, g, w, h0, cu)
        return (y * dy).sum() + (ht * dht).sum()

    grads = O.scan_bwd(v, g, w, h0, dy, dht, cu)
    for x, dx in zip((v, g, w, h0), grads):
        if x is not None:
            assert np.abs(differences(loss, x) - dx).max() < TOL


@pytest.mark.parametrize("temperature", [1.0, 0.6])
def test_logprob_gradients_are_the_differences(temperature):
    rng = np.random.default_rng(4)
    x = 2 * rng.standard_normal((4, 9))
    ids = np.array([3, -100, 0, 8])
    dlogp, dent = rng.standard_normal(4), rng.standard_normal(4)

    def loss():
        logp, ent, _ = O.token_logprobs(x, ids, temperature)
        return (logp * dlogp).sum() + (ent * dent).sum()

    dx = O.token_logprobs_bwd(x, ids, dlogp, dent, temperature)
    assert np.abs(differences(loss, x) - dx).max() < TOL
