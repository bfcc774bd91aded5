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


def sample_token(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Index taken from one row of logits by the uniform number u; -1 without a
    distribution."""
    x = np.asarray(x, dtype=np.float64)
    if np.isnan(x).any() or x.max() in (np.inf, -np.inf):
        return -1
    order, top_k = np.argsort(-x, kind="stable"), int(top_k)
    if temperature <= 0 or top_p <= 0 or top_k == 1:
        return int(order[0])
    w = np.exp((x - x.max()) / temperature)
    n = int(np.isfinite(x).sum())
    if min_p > 0:
        n = max(1, int((w >= min(min_p, 1.0)).sum()))
    if top_k > 0:
        n = min(n, top_k)
    if top_p < 1:
        mass = np.concatenate([[0.0], np.cumsum(w[order[:n]])])
        n = max(1, int((mass[:-1] < top_p * mass[-1]).sum()))
    kept = np.zeros_like(w)
    kept[order[:n]] = w[order[:n]]
    run = np.cumsum(kept)
    above = np.nonzero(run > min(max(u, 0.0), 1.0) * run[-1])[0]
    return int(above[0]) if above.size else int(np.nonzero(kept)[0][-1])


def softplus(v):
    return np.maximum(v, 0) + np.log1p(np.exp(-np.abs(v)))


def _selective(x, dt, A, B, C, D, z, bias, plus, h0, cu):
    """Inputs of the selective scan with its defaults filled in, B and C for each
    channel [B, T, D, N]."""
    nb, T, d = x.shape
    pre = dt if bias is None else dt + bias
    delta = softplus(pre) if plus else pre
    if B.ndim == 3:
        B, C = B[:, :, None], C[:, :, None]
    wide = lambda v: np.repeat(v, d // v.shape[2], axis=2)
    seqs = _sequences(nb, T, cu)
    h0 = np.zeros((len(seqs), d, A.shape[1])) if h0 is None else np.array(h0, dtype=np.float64)
    skip = np.zeros(d) if D is None else D
    return pre, delta, wide(B), wide(C), skip, seqs, h0


def selective_fwd(x, dt, A, B, C, D=None, z=None, bias=None, plus=False, h0=None, cu=None):
    """(y, states after every token, final states) of the selective state space scan."""
    _, delta, Bw, Cw, skip, seqs, ht = _selective(x, dt, A, B, C, D, z, bias, plus, h0, cu)
    H = np.zeros((*x.shape, A.shape[1]))
    for n, (b, lo, hi) in enumerate(seqs):
        h = ht[n].copy()
        for t in range(lo, hi):
            h = np.exp(delta[b, t][:, None] * A) * h + (delta[b, t] * x[b, t])[:, None] * Bw[b, t]
            H[b, t] = h
        ht[n] = h
    y = (H * Cw).sum(-1) + skip * x
    return (y if z is None else y * z / (1 + np.exp(-z))), H, ht


def selective_bwd(x, dt, A, B, C, D, z, bias, plus, h0, dy, dht=None, cu=None):
    """Gradients of sum(y dy) + sum(ht dht): a dict by the names of the inputs."""
    pre, delta, Bw, Cw, skip, seqs, start = _selective(x, dt, A, B, C, D, z, bias, plus, h0, cu)
    _, H, _ = selective_fwd(x, dt, A, B, C, D, z, bias, plus, h0, cu)
    sig = np.ones_like(x) if z is None else 1 / (1 + np.exp(-z))
    out = dy if z is None else dy * z * sig
    E, P = np.zeros_like(H), np.zeros_like(H)  # gradients of the states; decayed states
    dh0 = np.zeros_like(start) if dht is None else np.array(dht, dtype=np.float64)
    for n, (b, lo, hi) in enumerate(seqs):
        c = dh0[n].copy()
        for t in range(hi - 1, lo - 1, -1):
            a = np.exp(delta[b, t][:, None] * A)
            E[b, t] = out[b, t][:, None] * Cw[b, t] + c
            P[b, t] = a * (H[b, t - 1] if t > lo else start[n])
            c = a * E[b, t]
        dh0[n] = c
    sb = (E * Bw).sum(-1)
    ddelta = (E * P * A).sum(-1) + x * sb
    dpre = ddelta / (1 + np.exp(-pre)) if plus else ddelta
    groups = 1 if B.ndim == 3 else B.shape[2]
    fold = lambda v: v.reshape(*x.shape[:2], groups, -1, A.shape[1]).sum(3).reshape(B.shape)
    g = dict(x=delta * sb + skip * out, dt=dpre, A=(E * P * delta[..., None]).sum((0, 1)),
             B=fold(E * (delta * x)[..., None]), C=fold(H * out[..., None]), D=(out * x).sum((0, 1)),
             dt_bias=dpre.sum((0, 1)), h0=dh0)
    if z is not None:
        g["z"] = dy * ((H * Cw).sum(-1) + skip * x) * sig * (1 + z * (1 - sig))
    return g
