"""Float64 numpy oracle of the operators around the GDN-2 mixer: the gated
linear recurrence, token log probabilities and the AdamW step, each written
row by row from its definition."""

from __future__ import annotations

import numpy as np


def _sequences(B, T, cu):
    """(batch entry, first row, end row) of each sequence."""
    if cu is None:
        return [(b, 0, T) for b in range(B)]
    return [(0, int(cu[n]), int(cu[n + 1])) for n in range(len(cu) - 1)]


def scan_fwd(v, g, w=None, h0=None, cu=None):
    """h_t = exp(g_t) h_{t-1} + w_t v_t over [B, T, D]; returns (h, ht)."""
    B, T, D = v.shape
    seqs = _sequences(B, T, cu)
    y = np.zeros((B, T, D))
    ht = np.zeros((len(seqs), D)) if h0 is None else np.array(h0, dtype=np.float64)
    for n, (b, lo, hi) in enumerate(seqs):
        h = ht[n].copy()
        for t in range(lo, hi):
            h = np.exp(g[b, t]) * h + (v[b, t] if w is None else w[b, t] * v[b, t])
            y[b, t] = h
        ht[n] = h
    return y, ht


def scan_bwd(v, g, w, h0, dy, dht=None, cu=None):
    """Gradients (dv, dg, dw or None, dh0) of sum(y dy) + sum(ht dht)."""
    B, T, D = v.shape
    seqs = _sequences(B, T, cu)
    y, _ = scan_fwd(v, g, w, h0, cu)
    dv, dg = np.zeros_like(y), np.zeros_like(y)
    dw = None if w is None else np.zeros_like(y)
    dh0 = np.zeros((len(seqs), D))
    for n, (b, lo, hi) in enumerate(seqs):
        c = np.zeros(D) if dht is None else np.array(dht[n], dtype=np.float64)
        for t in range(hi - 1, lo - 1, -1):
            dh = dy[b, t] + c
            prev = y[b, t - 1] if t > lo else (np.zeros(D) if h0 is None else h0[n])
            a = np.exp(g[b, t])
            dg[b, t] = a * prev * dh
            dv[b, t] = dh if w is None else w[b, t] * dh
            if w is not None:
                dw[b, t] = v[b, t] * dh
            c = a * dh
        dh0[n] = c
    return dv, dg, dw, dh0


def token_logprobs(x, ids, temperature=1.0, ignore=-100):
    """Per row of x [R, V]: (log p of the id, entropy, log p of every token)."""
    R, V = x.shape
    logp, ent, table = np.zeros(R), np.zeros(R), np.full((R, V), -np.inf)
    for r in range(R):
        z = x[r] / temperature
        m = z.max()
        if m == -np.inf:
            logp[r] = 0.0 if ids[r] == ignore else -np.inf
            continue
        table[r] = z - m - np.log(np.exp(z - m).sum())
        if ids[r] == ignore:
            continue
        logp[r] = table[r, ids[r]]
        p = np.exp(table[r])
        ent[r] = -sum(p[j] * table[r, j] for j in range(V) if p[j] > 0)
    return logp, ent, table


def token_logprobs_bwd(x, ids, dlogp, dent=None, temperature=1.0, ignore=-100):
    """Gradient of sum(logp dlogp) + sum(entropy dent) with respect to x."""
    _, ent, table = token_logprobs(x, ids, temperature, ignore)
    dx = np.zeros_like(x)
    for r in range(x.shape[0]):
        if ids[r] == ignore or not np.isfinite(table[r]).any():
            continue
        p = np.exp(table[r])
        dx[r] = -dlogp[r] * p
        dx[r, ids[r]] += dlogp[r]
        if dent is not None:
            dx[r] -= dent[r] * p * np.where(p > 0, np.where(p > 0, table[r], 0.0) + ent[r], 0.0)
    return dx / temperature


def top_tokens(x, k):
    """Indices of the k largest of each row, equal values by rising index."""
    return np.argsort(-x, axis=1, kind="stable")[:, :k]


def e4m3(u):
    """u rounded to the nearest e4m3 value (ties to even); |u| <= 448."""
    step = 2.0 ** (np.floor(np.log2(np.maximum(np.abs(u), 2.0 ** -6))) - 3)
    return np.round(u / step) * step


def encode8(x, nonzero=False, block=256):
    """(codes, scales) of a flat array: x ~ codes * scale of its block."""
    codes, scales = np.zeros(x.size), np.zeros(-(-x.size // block))
    for b in range(scales.size):
        part = x[b * block:(b + 1) * block]
        most = np.abs(part).max()
        if most <= 1e-30:
            continue
        q = e4m3(part * (448.0 / most))
        if nonzero:
            q[(part > 0) & (q == 0)] = 2.0 ** -9
        codes[b * block:(b + 1) * block] = q
        scales[b] = most / 448.0
    return codes, scales


def adamw(p, g, m, v, step, lr, b1, b2, eps, wd):
    """(p, m, v) after one step."""
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    mhat, vhat = m / (1 - b1 ** step), v / (1 - b2 ** step)
    return p - lr * wd * p - lr * mhat / (np.sqrt(vhat) + eps), m, v
