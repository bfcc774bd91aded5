"""Cases of the operators around a training step, a prompt and a served token.

Three operators that a decoder built on the GDN-2 mixer runs next to it:

* the selective state space scan (``selective_scan``, ``selective_scan_step``):
  ``h_t = exp(dt_t A) h_{t-1} + dt_t x_t B_t``, ``y_t = (h_t C_t + D x_t) silu(z_t)``
  with a decay for each channel and state, over whole sequences with its
  gradient and for single tokens on a state pool;
* the choice of a token from logits and one given random number for each row
  (``sample_tokens``), with temperature, top-k, top-p and min-p;
* the norm of many gradients, the coefficient that clips it (``grad_norm``) and
  the clipping itself (``clip_grad_norm_``).

``listed()`` and ``draw()`` give the cases, ``prepare()`` a case's inputs,
``run()`` one pass (``own`` false: elementary torch operations; ``own`` true: the
framework's operators), ``work()`` the bytes and operations a pass cannot do
without, ``exact()`` the outputs in 64 bits.
"""

import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
SLAB = 1 << 28  # values of one temporary of the plain scan


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one decode step of 64 requests through a state pool (4096 = twice the hidden
        # size of the 24-layer decoder): latency of a serving step
        dict(name="sel_step_64", op="sel_step", n=64, pool=96, d=4096, n_state=16, groups=1,
             dtype="bf16", dtdtype="bf16", gate=True),
        # prefill of a packed ragged batch with empty and one-token requests, channels
        # that fill no whole tile, both states
        dict(name="sel_prefill_ragged", op="sel", b=1, t=9001, d=1000, n_state=16, groups=1, seqs=23,
             dtype="fp16", dtdtype="fp32", gate=False, train=False),
        # training: the mixer's config-1 token count at the decoder's width
        dict(name="sel_train_8x4096", op="sel", b=8, t=4096, d=2048, n_state=16, groups=1, seqs=0,
             dtype="bf16", dtdtype="bf16", gate=True, train=True),
        # training on one long sequence: few channels, the time axis has to be split
        dict(name="sel_train_65536", op="sel", b=1, t=65536, d=512, n_state=16, groups=1, seqs=0,
             dtype="bf16", dtdtype="bf16", gate=True, train=True),
        # training in 32 bits on packed documents, fewer states, two groups of channels
        # with their own input and output vectors
        dict(name="sel_train_packed_fp32", op="sel", b=1, t=6001, d=770, n_state=8, groups=2,
             seqs=11, dtype="fp32", dtdtype="fp32", gate=False, train=True),
        # a few rows of a small vocabulary in 32 bits, every option, each row its own:
        # latency of the smallest call
        dict(name="sample_3x1000", op="sample", rows=3, vocab=1000, dtype="fp32", top_k=True,
             top_p=True, min_p=True, masked=7),
        # one serving step of 64 requests, each with its own temperature, top-k and top-p
        dict(name="sample_serve_64", op="sample", rows=64, vocab=151936, dtype="bf16", top_k=True,
             top_p=True, min_p=False, masked=267),
        # 256 rollouts sampled by temperature alone, as a policy is: every token counts
        dict(name="sample_rollout_256", op="sample", rows=256, vocab=151936, dtype="bf16",
             top_k=False, top_p=False, min_p=False, masked=0),
        # 500 requests on an odd vocabulary: top-p and min-p without a top-k bound
        dict(name="sample_odd_500", op="sample", rows=500, vocab=32003, dtype="fp16", top_k=False,
             top_p=True, min_p=True, masked=3),
        # a small model's gradients, all in 32 bits: launch cost over many tensors
        dict(name="norm_small", op="norm", hidden=96, mlp=257, layers=3, vocab=503, dtype="fp32",
             wide_norms=False, kind="2", clip=False),
        # two layers of the decoder, clipped in place
        dict(name="clip_layers", op="norm", hidden=2048, mlp=5632, layers=2, vocab=1000, dtype="bf16",
             wide_norms=False, kind="2", clip=True),
        # embedding and two layers, the vectors' gradients in 32 bits: the norm and the
        # coefficient that the optimizer's step takes
        dict(name="norm_decoder", op="norm", hidden=2048, mlp=5632, layers=2, vocab=151936,
             dtype="bf16", wide_norms=True, kind="2", clip=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("sel_step", "sel", "sel", "sample", "sample", "norm"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    if op in ("sel", "sel_step"):
        n_state, groups = rng.choice((16, 16, 16, 8, 32, rng.randrange(1, 65))), rng.choice((1, 1, 1, 2, 4))
        kind = dict(n_state=n_state, groups=groups, dtype=dtype, dtdtype=rng.choice((dtype, dtype, "fp32")),
                    gate=rng.random() < 0.5)
        if op == "sel_step":
            n = _log_int(rng, 1, 512)
            return dict(op=op, n=n, pool=n + rng.randrange(64), d=groups * _log_int(rng, 16, 2048), **kind)
        d, t = groups * _log_int(rng, 8, 1024), _log_int(rng, 1, 65536)
        room = 1_000_000_000 // (d * n_state)
        t = max(1, min(t, room))
        b = max(1, min(room // t, _log_int(rng, 1, 64)))
        seqs = rng.choice((0, 0, _log_int(rng, 2, 64)))
        return dict(op=op, b=1 if seqs else b, t=t, d=d, seqs=seqs, train=rng.random() < 0.6, **kind)
    if op == "sample":
        vocab = _log_int(rng, 100, 160000)
        return dict(op=op, rows=min(_log_int(rng, 1, 2048), 39_000_000 // vocab), vocab=vocab, dtype=dtype,
                    top_k=rng.random() < 0.5, top_p=rng.random() < 0.5, min_p=rng.random() < 0.3,
                    masked=rng.choice((0, vocab // 50)))
    hidden = _log_int(rng, 32, 2048)
    return dict(op=op, hidden=hidden, mlp=int(hidden * rng.uniform(1.5, 3.5)), layers=rng.randrange(1, 4),
                vocab=_log_int(rng, 100, 60000), dtype=dtype, wide_norms=rng.random() < 0.5,
                kind=rng.choice(("2", "2", "inf")), clip=rng.random() < 0.5)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _lengths(total, n):
    """``n`` ragged lengths that add up to ``total``, one of them 0 and one of them 1."""
    rng = random.Random(1000003 * total + n)
    cuts = sorted(rng.randrange(total + 1) for _ in range(n - 1))
    if n >= 3:
        cuts[n // 2] = cuts[n // 2 - 1]
    if n >= 5 and total:
        cuts[0] = 1
        cuts.sort()
    ends = [0] + cuts + [total]
    return [b - a for a, b in zip(ends, ends[1:])]


def _shapes(c):
    """Gradient shapes of a decoder with the mixer in each layer: projections, two
    low-rank gates, three short convolutions, norms, decays and a gated MLP."""
    h, m = c["hidden"], c["mlp"]
    r = max(1, h // 16)
    layer = [(h, h)] * 6 + [(r, h), (h, r)] * 2 + [(h,)] * 4 + [(h, 1, 4)] * 3 + [(r,), (max(1, h // 128),)]
    layer += [(m, h), (m, h), (h, m)]
    return [(c["vocab"], h)] + layer * c["layers"] + [(h,)]


def _rand(gen, *shape, lo=0.0, hi=1.0):
    return torch.empty(shape, device=DEV).uniform_(lo, hi, generator=gen)


def _randn(gen, *shape, dtype=torch.float32, scale=1.0, shift=0.0):
    x = torch.empty(shape, dtype=dtype, device=DEV)
    x.normal_(shift, scale, generator=gen)
    return x


def _prepare_sel(c, gen):
    dt, d, n = DTYPES[c["dtype"]], c["d"], c["n_state"]
    step = c["op"] == "sel_step"
    lead = (c["n"],) if step else (c["b"], c["t"])
    vec = lead + ((c["groups"], n) if c["groups"] > 1 else (n,))
    s = dict(case=c)
    # what the short convolution and its SiLU leave
    s["x"] = torch.nn.functional.silu(_randn(gen, *lead, d)).to(dt)
    # time steps before their softplus: their bias spreads them over 0.001 .. 0.1
    s["dt"] = _randn(gen, *lead, d, scale=0.5).to(DTYPES[c["dtdtype"]])
    target = torch.exp(_rand(gen, d, lo=math.log(1e-3), hi=math.log(0.1)))
    s["dt_bias"] = target + torch.log(-torch.expm1(-target))
    s["A"] = -torch.arange(1.0, n + 1, device=DEV) * torch.exp(_randn(gen, d, n, scale=0.1))
    s["B"], s["C"] = _randn(gen, *vec, dtype=dt), _randn(gen, *vec, dtype=dt)
    s["D"] = _randn(gen, d, scale=0.2, shift=1.0)
    s["z"] = _randn(gen, *lead, d, dtype=dt) if c["gate"] else None
    if step:
        s["slots"] = torch.randperm(c["pool"], generator=gen, device=DEV)[: c["n"]].to(torch.int32)
        s["pool"] = _randn(gen, c["pool"], d, n, scale=0.3)
        return s
    lens = _lengths(c["t"], c["seqs"]) if c["seqs"] else [c["t"]] * c["b"]
    s["longest"], s["lens"] = max(lens), lens
    s["cu"] = torch.tensor([0] + lens, dtype=torch.int32).cumsum(0, dtype=torch.int32).to(DEV)
    s["h0"] = _randn(gen, len(lens), d, n, scale=0.3)
    if c["train"]:
        s["dy"], s["dht"] = _randn(gen, *lead, d, dtype=dt), _randn(gen, len(lens), d, n)
        for k in LEAVES:
            if s[k] is not None:
                s[k].requires_grad_()
    return s


LEAVES = ("x", "dt", "A", "B", "C", "D", "z", "dt_bias", "h0")


def _prepare_sample(c, gen):
    n, vocab = c["rows"], c["vocab"]
    logits = _randn(gen, n, vocab, dtype=DTYPES[c["dtype"]], scale=2.5)
    rows = torch.arange(n, device=DEV)
    for lift in (9.0, 7.0, 6.0):  # a trained model prefers a few tokens
        logits[rows, torch.randint(0, vocab, (n,), generator=gen, device=DEV)] += lift
    if c["masked"]:
        logits[:, vocab - c["masked"]:] = -math.inf
    # options of each request; some rows have an option off (0 or 1)
    off = lambda: _rand(gen, n) < 0.2  # noqa: E731
    s = dict(case=c, logits=logits, uniform=_rand(gen, n), temperature=_rand(gen, n, lo=0.5, hi=1.3))
    s["top_k"] = (torch.randint(1, 200, (n,), generator=gen, device=DEV).masked_fill(off(), 0).to(torch.int32)
                  if c["top_k"] else None)
    s["top_p"] = _rand(gen, n, lo=0.5, hi=0.99).masked_fill(off(), 1.0) if c["top_p"] else None
    s["min_p"] = _rand(gen, n, lo=0.001, hi=0.1).masked_fill(off(), 0.0) if c["min_p"] else None
    return s


def _prepare_norm(c, gen):
    dt = DTYPES[c["dtype"]]
    grads = []
    for sh in _shapes(c):
        wide = c["wide_norms"] and len(sh) == 1
        grads.append(_randn(gen, *sh, dtype=torch.float32 if wide else dt, scale=1e-3))
    return dict(case=c, grads=grads, limit=0.5 * 1e-3 * math.sqrt(sum(g.numel() for g in grads)))


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    make = {"sample": _prepare_sample, "norm": _prepare_norm}.get(case["op"], _prepare_sel)
    return make(case, gen)


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _scan_rows(a, x, longest):
    """h_r = a_r h_{r-1} + x_r down the rows by doubling spans; overwrites both."""
    span = 1
    while span < longest:
        x[span:] += a[span:] * x[:-span]
        a[span:] = a[span:] * a[:-span]
        span *= 2
    return x


def _softplus(v):
    return v.clamp(min=0) + torch.log1p(torch.exp(-v.abs()))


def _per_channel(v, rows, c, n0, n1):
    """States n0 .. n1 of the groups' vectors as [rows, groups, 1, n]."""
    return v.detach().reshape(rows, c["groups"], 1, -1)[..., n0:n1].float()


def _plain_sel(s):
    c = s["case"]
    shape, d, g, n = s["x"].shape, c["d"], c["groups"], c["n_state"]
    rows, w = shape[0] * shape[1], d // g
    flat = lambda v: v.detach().reshape(rows, g, w).float()  # noqa: E731
    par = lambda v: v.detach().view(1, g, w)  # noqa: E731
    x, pre = flat(s["x"]), flat(s["dt"]) + par(s["dt_bias"])
    dt = _softplus(pre)
    dtx = dt * x
    cu = s["cu"].long()
    full = (cu[1:] > cu[:-1]).nonzero().flatten()
    first, last = cu[full], cu[full + 1] - 1
    h0 = s["h0"].detach()
    ht = h0.clone()
    gate = z = None
    if c["gate"]:
        z = flat(s["z"])
        gate = torch.sigmoid(z)
    out_sum = torch.zeros_like(x)
    train = c["train"]
    if train:
        dy = flat(s["dy"])
        dout = dy * (z * gate) if c["gate"] else dy
        s_b, s_a = torch.zeros_like(x), torch.zeros_like(x)
        dht = s["dht"]
        dh0, dA = dht.clone(), torch.empty_like(h0[0])
        dB, dC = torch.empty(rows, g, n, device=DEV), torch.empty(rows, g, n, device=DEV)
    slab = max(1, SLAB // (rows * d))
    for n0 in range(0, n, slab):
        n1 = min(n0 + slab, n)
        A = s["A"].detach()[:, n0:n1].view(1, g, w, n1 - n0)
        B, C = _per_channel(s["B"], rows, c, n0, n1), _per_channel(s["C"], rows, c, n0, n1)
        a = torch.exp(dt[..., None] * A)
        v = dtx[..., None] * B
        start = h0[full][..., n0:n1].reshape(-1, g, w, n1 - n0)
        v[first] += a[first] * start
        kept = a.clone()
        kept[first] = 0.0
        h = _scan_rows(kept.clone(), v, s["longest"])
        ht[full, :, n0:n1] = h[last].reshape(-1, d, n1 - n0)
        out_sum += (h * C).sum(-1)
        if not train:
            continue
        e = dout[..., None] * C
        dC[..., n0:n1] = (dout[..., None] * h).sum(2)
        e[last] += dht[full][..., n0:n1].reshape(-1, g, w, n1 - n0)
        after = torch.zeros_like(a)
        after[:-1] = kept[1:]
        dh = _scan_rows(after.flip(0), e.flip(0), s["longest"]).flip(0)
        del after, e, kept
        dB[..., n0:n1] = (dtx[..., None] * dh).sum(2)
        s_b += (dh * B).sum(-1)
        dh0[full, :, n0:n1] = (a[first] * dh[first]).reshape(-1, d, n1 - n0)
        before = torch.zeros_like(h)
        before[1:] = h[:-1]
        before[first] = start
        q = a * before * dh
        del before, h, dh, a
        s_a += (q * A).sum(-1)
        dA[:, n0:n1] = (dt[..., None] * q).sum(0).reshape(d, n1 - n0)
    skip = out_sum + par(s["D"]) * x
    y = skip * (z * gate) if c["gate"] else skip
    like = lambda v, t: v.reshape(t.shape).to(t.dtype)  # noqa: E731
    out = dict(y=like(y, s["x"]), ht=ht)
    if train:
        ddt = (s_a + x * s_b) * torch.sigmoid(pre)
        out.update(dx=like(dt * s_b + par(s["D"]) * dout, s["x"]), ddt=like(ddt, s["dt"]), dA=dA,
                   dB=like(dB, s["B"]), dC=like(dC, s["C"]), dD=(dout * x).sum(0).view(d),
                   ddt_bias=ddt.sum(0).view(d), dh0=dh0)
        if c["gate"]:
            out["dz"] = like(dy * skip * gate * (1 + z * (1 - gate)), s["z"])
    return out


def _plain_sel_step(s):
    c = s["case"]
    rows, g, d = c["n"], c["groups"], c["d"]
    flat = lambda v: v.reshape(rows, g, d // g).float()  # noqa: E731
    x = flat(s["x"])
    dt = _softplus(flat(s["dt"]) + s["dt_bias"].view(1, g, -1))
    at = s["slots"].long()
    old = s["pool"][at].view(rows, g, d // g, -1)
    h = torch.exp(dt[..., None] * s["A"].view(1, g, d // g, -1)) * old
    h = h + (dt * x)[..., None] * _per_channel(s["B"], rows, c, 0, None)
    y = (h * _per_channel(s["C"], rows, c, 0, None)).sum(-1) + s["D"].view(1, g, -1) * x
    if c["gate"]:
        z = flat(s["z"])
        y = y * z * torch.sigmoid(z)
    s["pool"][at] = h.view(rows, d, -1)
    return dict(y=y.view(rows, d).to(s["x"].dtype), pool=s["pool"])


def _order_keys(x):
    """Whole numbers that fall as values do, equal values by rising index."""
    bits = (x.float() + 0.0).view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    return order * (1 << 32) + ((1 << 31) - 1 - torch.arange(x.shape[1], device=DEV))


def _plain_sample(s):
    """In 64 bits: a token's running sum decides against its neighbours' by the last digits."""
    c = s["case"]
    z = s["logits"].double() / s["temperature"].double()[:, None]
    w = torch.exp(z - z.amax(1, keepdim=True))
    if c["min_p"]:
        w = torch.where(w >= s["min_p"].double()[:, None], w, 0.0)
    if c["top_k"] or c["top_p"]:
        at = _order_keys(s["logits"]).sort(1, descending=True).indices
        v = w.gather(1, at)
        if c["top_k"]:
            k = s["top_k"].long()
            k = torch.where(k > 0, k, c["vocab"])[:, None]
            v = torch.where(torch.arange(c["vocab"], device=DEV) < k, v, 0.0)
        if c["top_p"]:
            p = s["top_p"].double()[:, None]
            total = v.cumsum(1)
            v = torch.where((p >= 1) | (total - v < p * total[:, -1:]), v, 0.0)
        w = torch.zeros_like(w).scatter_(1, at, v)
    total = w.cumsum(1)
    return (total <= s["uniform"].double()[:, None] * total[:, -1:]).sum(1)


def _coefficient(norm, limit):
    return torch.where(torch.isfinite(norm), (limit / (norm + 1e-6)).clamp(max=1.0), 1.0)


def _plain_norm(s):
    c = s["case"]
    if c["clip"]:  # a limit that falls a little, so that every pass has something to clip
        s["limit"] *= 0.995
    if c["kind"] == "2":
        norm = torch.stack([g.double().square().sum() for g in s["grads"]]).sum().sqrt().float()
    else:
        norm = torch.stack([g.abs().amax().float() for g in s["grads"]]).amax()
    coef = _coefficient(norm, s["limit"])
    out = dict(norm=norm, coef=coef, found_inf=(~torch.isfinite(norm)).float())
    if c["clip"]:
        for g in s["grads"]:
            g.copy_(g.float() * coef)
        out["grads"] = s["grads"]
    return out


# ---------------------------------------------------------------------------
# the framework's operators
# ---------------------------------------------------------------------------
def _own_sel(s):
    from qwendopamine_b200 import selective_scan

    c = s["case"]
    y, ht = selective_scan(s["x"], s["dt"], s["A"], s["B"], s["C"], s["D"], s["z"], dt_bias=s["dt_bias"],
                           dt_softplus=True, initial_state=s["h0"], output_final_state=True,
                           cu_seqlens=s["cu"] if c["seqs"] else None)
    out = dict(y=y.detach(), ht=ht.detach())
    if c["train"]:
        names = [k for k in LEAVES if s[k] is not None]
        grads = torch.autograd.grad((y, ht), [s[k] for k in names], (s["dy"], s["dht"]))
        out.update(("d" + k, v) for k, v in zip(names, grads))
    return out


def _own_sel_step(s):
    from qwendopamine_b200 import selective_scan_step

    y = selective_scan_step(s["x"], s["dt"], s["A"], s["B"], s["C"], s["D"], s["z"], dt_bias=s["dt_bias"],
                            dt_softplus=True, state=s["pool"], state_indices=s["slots"])
    return dict(y=y, pool=s["pool"])


def _own_sample(s):
    from qwendopamine_b200 import sample_tokens

    options = {k: s[k] for k in ("top_k", "top_p", "min_p") if s[k] is not None}
    return sample_tokens(s["logits"], s["uniform"], temperature=s["temperature"], **options)


def _own_norm(s):
    from qwendopamine_b200 import clip_grad_norm_, grad_norm

    c = s["case"]
    kind = float(c["kind"])
    if c["clip"]:
        s["limit"] *= 0.995
        r = clip_grad_norm_(s["grads"], s["limit"], norm_type=kind)
        return dict(norm=r.norm, coef=r.clip_coef, found_inf=r.found_inf, grads=s["grads"])
    r = grad_norm(s["grads"], max_norm=s["limit"], norm_type=kind)
    return dict(norm=r.norm, coef=r.clip_coef, found_inf=r.found_inf)


def run(state):
    op = state["case"]["op"]
    if own:
        return {"sel": _own_sel, "sel_step": _own_sel_step, "sample": _own_sample,
                "norm": _own_norm}[op](state)
    with torch.no_grad():
        return {"sel": _plain_sel, "sel_step": _plain_sel_step, "sample": _plain_sample,
                "norm": _plain_norm}[op](state)


# ---------------------------------------------------------------------------
# work and exact values
# ---------------------------------------------------------------------------
def work(case):
    c = case
    e = SIZE[c["dtype"]]
    if c["op"] in ("sel", "sel_step"):
        d, n, gate = c["d"], c["n_state"], c["gate"]
        rows = c["n"] if c["op"] == "sel_step" else c["b"] * c["t"]
        states = 4 * d * n * (c["n"] if c["op"] == "sel_step" else c["seqs"] or c["b"])
        ins = rows * (d * (e + SIZE[c["dtdtype"]] + e * gate) + 2 * e * c["groups"] * n) + 4 * d * (n + 2)
        # a decay (one product, one exponential) and three products and sums for each state
        flops = rows * d * (7 * n + 8)
        if c["op"] == "sel" and c["train"]:
            return dict(bytes=2 * ins + 2 * e * rows * d + 4 * states, flops=flops + rows * d * (18 * n + 12))
        return dict(bytes=ins + e * rows * d + 2 * states, flops=flops)
    if c["op"] == "sample":
        n = c["rows"] * c["vocab"]
        return dict(bytes=n * e + c["rows"] * (16 + 4 * (c["top_k"] + c["top_p"] + c["min_p"])),
                    flops=n * 4)
    sizes = [(math.prod(sh), 4 if c["wide_norms"] and len(sh) == 1 else e) for sh in _shapes(c)]
    total = sum(k * b for k, b in sizes)
    return dict(bytes=total * (2 if c["clip"] else 1), flops=(3 if c["clip"] else 2) * sum(k for k, _ in sizes))


def _exact_sel(s):
    """Token by token from the definition; the sums over rows a slab of rows at a time."""
    c = s["case"]
    bsz, t_all = s["x"].shape[:2]
    rows, d, n, g = bsz * t_all, c["d"], c["n_state"], c["groups"]
    wide = lambda v: v.detach().double()  # noqa: E731
    x, dt_in = wide(s["x"]).reshape(rows, d), wide(s["dt"]).reshape(rows, d)
    pre = dt_in + wide(s["dt_bias"])
    dt = torch.logaddexp(pre, torch.zeros_like(pre))
    A, D, h0 = wide(s["A"]), wide(s["D"]), wide(s["h0"])
    Bv, Cv = (wide(s[k]).reshape(rows, g, n) for k in ("B", "C"))
    chan = lambda v: v.repeat_interleave(d // g, dim=-2)  # noqa: E731  [.., g, n] -> [.., d, n]
    if c["seqs"]:
        ends = s["cu"].tolist()
        runs = [(k, torch.arange(lo, hi, device=DEV)[None]) for k, (lo, hi) in enumerate(zip(ends, ends[1:]))]
        runs = [(slice(k, k + 1), r) for k, r in runs]
    else:
        runs = [(slice(0, bsz), torch.arange(rows, device=DEV).view(bsz, t_all))]
    H = torch.empty(rows, d, n, dtype=torch.float64, device=DEV)
    ht = h0.clone()
    for who, r in runs:
        h = h0[who]
        for t in range(r.shape[1]):
            i = r[:, t]
            h = torch.exp(dt[i][..., None] * A) * h + (dt[i] * x[i])[..., None] * chan(Bv[i])
            H[i] = h
        ht[who] = h
    slabs = [slice(lo, min(lo + max(1, (1 << 27) // (d * n)), rows))
             for lo in range(0, rows, max(1, (1 << 27) // (d * n)))]
    core = torch.empty(rows, d, dtype=torch.float64, device=DEV)
    for sl in slabs:
        core[sl] = torch.einsum("rgwn,rgn->rgw", H[sl].view(-1, g, d // g, n), Cv[sl]).reshape(-1, d)
    skip = core + D * x
    z = wide(s["z"]).reshape(rows, d) if c["gate"] else None
    silu = z / (1 + torch.exp(-z)) if c["gate"] else torch.ones_like(x)
    shaped = lambda v, k: v.reshape(s[k].shape)  # noqa: E731
    out = dict(y=shaped(skip * silu, "x"), ht=ht)
    if not c["train"]:
        return out
    dy, dht = wide(s["dy"]).reshape(rows, d), wide(s["dht"])
    dout = dy * silu
    G = torch.empty_like(H)  # gradient of every state
    dh0 = dht.clone()
    before = torch.empty_like(H)
    before[1:] = H[:-1]
    for who, r in runs:
        if not r.shape[1]:
            continue
        before[r[:, 0]] = h0[who]
        carry = dht[who]
        for t in range(r.shape[1] - 1, -1, -1):
            i = r[:, t]
            carry = carry + dout[i][..., None] * chan(Cv[i])
            G[i] = carry
            carry = torch.exp(dt[i][..., None] * A) * carry
        dh0[who] = carry
    dB, dC = torch.empty_like(Bv), torch.empty_like(Cv)
    dA = torch.zeros_like(A)
    ddt, sb = torch.empty_like(x), torch.empty_like(x)
    for sl in slabs:
        split = lambda v: v.view(-1, g, d // g, n)  # noqa: E731
        dB[sl] = torch.einsum("rgwn,rgw->rgn", split(G[sl]), (dt[sl] * x[sl]).view(-1, g, d // g))
        dC[sl] = torch.einsum("rgwn,rgw->rgn", split(H[sl]), dout[sl].view(-1, g, d // g))
        sb[sl] = torch.einsum("rgwn,rgn->rgw", split(G[sl]), Bv[sl]).reshape(-1, d)
        dlog = torch.exp(dt[sl][..., None] * A) * before[sl] * G[sl]  # gradient of dt A
        dA += torch.einsum("rdn,rd->dn", dlog, dt[sl])
        ddt[sl] = torch.einsum("rdn,dn->rd", dlog, A) + x[sl] * sb[sl]
    dpre = ddt / (1 + torch.exp(-pre))
    out.update(dx=shaped(dt * sb + D * dout, "x"), ddt=shaped(dpre, "dt"), dA=dA, dB=shaped(dB, "B"),
               dC=shaped(dC, "C"), dD=(dout * x).sum(0), ddt_bias=dpre.sum(0), dh0=dh0)
    if c["gate"]:
        sig = 1 / (1 + torch.exp(-z))
        out["dz"] = shaped(dy * skip * (sig + z * sig * (1 - sig)), "z")
    return out


def _exact_sel_step(s):
    c = s["case"]
    at = s["slots"].long()
    reps = c["d"] // c["groups"]
    vec = lambda k: s[k].double().view(c["n"], c["groups"], -1).repeat_interleave(reps, 1)  # noqa: E731
    x, pre = s["x"].double(), s["dt"].double() + s["dt_bias"].double()
    dt = torch.logaddexp(pre, torch.zeros_like(pre))
    pool = s["pool"].double()
    h = torch.exp(torch.einsum("bd,dn->bdn", dt, s["A"].double())) * pool[at]
    h = h + torch.einsum("bd,bdn->bdn", dt * x, vec("B"))
    y = torch.einsum("bdn,bdn->bd", h, vec("C")) + x * s["D"].double()
    if c["gate"]:
        z = s["z"].double()
        y = y * (z / (1 + torch.exp(-z)))
    pool[at] = h
    return dict(y=y, pool=pool)


def _exact_sample(s):
    """Row by row through a stable sort."""
    c = s["case"]
    ids = []
    for r in range(c["rows"]):
        p = torch.softmax(s["logits"][r].double() / s["temperature"][r].double(), 0)
        falling, at = torch.sort(s["logits"][r].float(), descending=True, stable=True)
        keep = torch.ones(c["vocab"], dtype=torch.bool, device=DEV)
        ranked = p[at]
        if c["min_p"]:
            keep &= ranked >= s["min_p"][r].double() * ranked[0]
        if c["top_k"] and int(s["top_k"][r]) > 0:
            keep[int(s["top_k"][r]):] = False
        ranked = ranked * keep
        if c["top_p"] and float(s["top_p"][r]) < 1:
            mass = torch.cumsum(ranked / ranked.sum(), 0)
            enough = int((mass < s["top_p"][r].double()).sum())
            ranked[enough + 1:] = 0
        chosen = torch.zeros_like(p)
        chosen[at] = ranked
        mass = torch.cumsum(chosen, 0)
        ids.append(torch.searchsorted(mass, s["uniform"][r].double() * mass[-1], right=True))
    return torch.stack(ids)


def _exact_norm(s):
    c = s["case"]
    limit = s["limit"] * 0.995 if c["clip"] else s["limit"]
    if c["kind"] == "2":
        norm = math.sqrt(math.fsum(float(torch.linalg.vector_norm(g, dtype=torch.float64)) ** 2
                                   for g in s["grads"]))
    else:
        norm = max(float(g.abs().max()) for g in s["grads"])
    coef = min(1.0, limit / (norm + 1e-6))
    one = lambda v: torch.tensor(v, dtype=torch.float64, device=DEV)  # noqa: E731
    out = dict(norm=one(norm), coef=one(coef), found_inf=one(0.0))
    if c["clip"]:
        out["grads"] = [g.double() * coef for g in s["grads"]]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"sel": _exact_sel, "sel_step": _exact_sel_step, "sample": _exact_sample,
            "norm": _exact_norm}[case["op"]](s)
