"""Cases of the training- and serving-step operators around the GDN-2 mixer.

Three operators that a decoder built on the mixer runs next to it:

* the gated linear recurrence ``h_t = exp(g_t) h_{t-1} + w_t v_t`` (``gated_scan``,
  ``gated_scan_step``), its gradient and its single-token form on a state pool;
* the log probabilities of given tokens with entropy and top alternatives
  (``token_logprobs``) and their gradient;
* the AdamW step over many tensors with 32-bit or 8-bit states (``adamw_step``).

``listed()`` and ``draw()`` give the cases, ``prepare()`` a case's inputs,
``run()`` one pass (``own`` false: elementary torch operations in 32 bits;
``own`` true: the framework's operators), ``work()`` the bytes and operations
a pass cannot do without, ``exact()`` the outputs in 64 bits.
"""

import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
IGNORE = -100
BLOCK = 256  # elements that share a scale in the 8-bit optimizer states
HYPER = dict(lr=3e-4, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1)


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one decode step of 64 requests through a state pool (2048 = hidden size of
        # the 24-layer decoder): latency of a serving step
        dict(name="scan_step_64", op="scan_step", n=64, pool=96, d=2048, dtype="bf16", gdtype="fp32",
             gate=True),
        # prefill of a packed ragged batch with empty and one-token requests, channels
        # that fill no whole tile, both states
        dict(name="scan_prefill_ragged", op="scan", b=1, t=9001, d=1000, seqs=23, dtype="fp16",
             gdtype="fp16", gate=False, train=False),
        # training: the mixer's config-1 token count at the decoder's width
        dict(name="scan_train_8x4096", op="scan", b=8, t=4096, d=2048, seqs=0, dtype="bf16",
             gdtype="fp32", gate=True, train=True),
        # training on one long sequence: few channels, the time axis has to be split
        dict(name="scan_train_131072", op="scan", b=1, t=131072, d=1024, seqs=0, dtype="bf16",
             gdtype="fp32", gate=False, train=True),
        # a few rows of a small vocabulary in 32 bits: latency of the smallest call
        dict(name="logp_3x1000", op="logp", rows=3, vocab=1000, dtype="fp32", top=20, entropy=True,
             temperature=1.0, masked=0, train=False),
        # one serving step of 32 requests: chosen token, entropy and five alternatives,
        # sampling temperature, padded vocabulary entries masked with -inf
        dict(name="logp_serve_32", op="logp", rows=32, vocab=151936, dtype="bf16", top=5,
             entropy=True, temperature=0.7, masked=267, train=False),
        # scoring 2048 prompt tokens with their best alternative
        dict(name="logp_score_2048", op="logp", rows=2048, vocab=151936, dtype="bf16", top=1,
             entropy=False, temperature=1.0, masked=0, train=False),
        # a training chunk of 4096 tokens: loss, entropy bonus and the logits' gradient
        dict(name="logp_train_4096", op="logp", rows=4096, vocab=151936, dtype="bf16", top=0,
             entropy=True, temperature=1.0, masked=0, train=True),
        # training with an odd vocabulary in 32 bits: rows start off any alignment
        dict(name="logp_train_odd", op="logp", rows=1501, vocab=32003, dtype="fp32", top=0,
             entropy=False, temperature=1.0, masked=3, train=True),
        # a small model's parameters, all in 32 bits: launch cost over many tensors
        dict(name="adamw_small", op="adamw", hidden=96, mlp=257, layers=3, vocab=503, dtype="fp32",
             bits=32, master=False),
        # two layers of the decoder in bf16 with 8-bit states
        dict(name="adamw_layers_8bit", op="adamw", hidden=2048, mlp=5632, layers=2, vocab=1000,
             dtype="bf16", bits=8, master=False),
        # embedding and two layers of the decoder in bf16 with 32-bit states and master weights
        dict(name="adamw_decoder_32bit", op="adamw", hidden=2048, mlp=5632, layers=2, vocab=151936,
             dtype="bf16", bits=32, master=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("scan_step", "scan", "scan", "logp", "logp", "adamw", "adamw"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    if op == "scan_step":
        n = _log_int(rng, 1, 1024)
        return dict(op=op, n=n, pool=n + rng.randrange(64), d=_log_int(rng, 32, 8192), dtype=dtype,
                    gdtype=rng.choice(("fp32", dtype)), gate=rng.random() < 0.5)
    if op == "scan":
        d, t = _log_int(rng, 16, 4096), _log_int(rng, 1, 131072)
        most = max(1, 120_000_000 // (d * t))
        b = min(most, _log_int(rng, 1, 64))
        if b * t * d > 120_000_000:
            t = max(1, 120_000_000 // d)
        seqs = rng.choice((0, 0, _log_int(rng, 2, 64)))
        return dict(op=op, b=1 if seqs else b, t=t, d=d, seqs=seqs, dtype=dtype,
                    gdtype=rng.choice(("fp32", dtype)), gate=rng.random() < 0.5,
                    train=rng.random() < 0.6)
    if op == "logp":
        vocab = _log_int(rng, 100, 160000)
        rows = min(_log_int(rng, 1, 8192), 300_000_000 // vocab)
        train = rng.random() < 0.5
        return dict(op=op, rows=rows, vocab=vocab, dtype=dtype, top=0 if train else rng.choice((0, 1, 5, 20)),
                    entropy=rng.random() < 0.5, temperature=rng.choice((1.0, 1.0, 0.7, 1.3)),
                    masked=rng.choice((0, vocab // 50)), train=train)
    hidden = _log_int(rng, 32, 2048)
    return dict(op=op, hidden=hidden, mlp=int(hidden * rng.uniform(1.5, 3.5)), layers=rng.randrange(1, 4),
                vocab=_log_int(rng, 100, 60000), dtype=rng.choice(("bf16", "fp16", "fp32")),
                bits=rng.choice((8, 32)), master=rng.random() < 0.4)


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
    """Parameter shapes of a decoder with the mixer in each layer: projections, two
    low-rank gates, three short convolutions, norms, decays and a gated MLP."""
    h, m = c["hidden"], c["mlp"]
    r = max(1, h // 16)
    layer = [(h, h)] * 6 + [(r, h), (h, r)] * 2 + [(h,)] * 4 + [(h, 1, 4)] * 3 + [(r,), (max(1, h // 128),)]
    layer += [(m, h), (m, h), (h, m)]
    return [(c["vocab"], h)] + layer * c["layers"] + [(h,)]


def _count(shape):
    return math.prod(shape)


def _randn(gen, *shape, dtype=torch.float32, scale=1.0, shift=0.0):
    x = torch.empty(shape, dtype=dtype, device=DEV)
    x.normal_(shift, scale, generator=gen)
    return x


def prepare(case, seed):
    c = case
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[c["dtype"]]
    if c["op"] in ("scan", "scan_step"):
        shape = (c["n"], c["d"]) if c["op"] == "scan_step" else (c["b"], c["t"], c["d"])
        v = _randn(gen, *shape, dtype=dt)
        g = torch.nn.functional.logsigmoid(_randn(gen, *shape, shift=3.0)).to(DTYPES[c["gdtype"]])
        w = torch.sigmoid(_randn(gen, *shape)).to(dt) if c["gate"] else None
        if c["op"] == "scan_step":
            slots = torch.randperm(c["pool"], generator=gen, device=DEV)[: c["n"]].to(torch.int32)
            return dict(case=c, v=v, g=g, w=w, pool=_randn(gen, c["pool"], c["d"]), slots=slots)
        lens = _lengths(c["t"], c["seqs"]) if c["seqs"] else [c["t"]] * c["b"]
        s = dict(case=c, v=v, g=g, w=w, h0=_randn(gen, len(lens), c["d"]), cu=None, longest=max(lens))
        cu = torch.tensor([0] + lens, dtype=torch.int32).cumsum(0, dtype=torch.int32)
        s["cu"] = cu.to(DEV)
        if c["train"]:
            s["dy"], s["dht"] = _randn(gen, *shape, dtype=dt), _randn(gen, len(lens), c["d"])
            for k in ("v", "g", "w", "h0"):
                if s[k] is not None:
                    s[k].requires_grad_()
        return s
    if c["op"] == "logp":
        n, vocab = c["rows"], c["vocab"]
        logits = _randn(gen, n, vocab, dtype=dt, scale=2.5)
        ids = torch.randint(0, vocab - c["masked"], (n,), generator=gen, device=DEV)
        rows = torch.arange(n, device=DEV)
        logits[rows, ids] += 6.0  # a trained model prefers the given token
        if c["masked"]:
            logits[:, vocab - c["masked"]:] = -math.inf
        s = dict(case=c, logits=logits, ids=ids)
        if c["train"]:
            ids[torch.rand(n, generator=gen, device=DEV) < 0.1] = IGNORE  # prompt tokens bear no loss
            s["dlogp"] = _randn(gen, n, scale=0.1, shift=-1.0) / n
            s["dent"] = torch.full((n,), -0.01 / n, device=DEV) if c["entropy"] else None
            logits.requires_grad_()
        return s
    # the optimizer: one flat buffer for each kind, every tensor a view that starts on
    # a whole block of it, as a training program with flat gradient buffers keeps them
    shapes = _shapes(c)
    starts, total = [], 0
    for sh in shapes:
        starts.append(total)
        total += -(-_count(sh) // BLOCK) * BLOCK

    def views(flat, per=1):
        if per == 1:
            return [flat[o: o + _count(sh)].view(sh) for o, sh in zip(starts, shapes)]
        return [flat[o // per: o // per + -(-_count(sh) // per)] for o, sh in zip(starts, shapes)]

    def padded(x):
        """Zeros between the tensors."""
        keep = torch.zeros(total, dtype=torch.bool, device=DEV)
        for o, sh in zip(starts, shapes):
            keep[o: o + _count(sh)] = True
        return x.mul_(keep)

    wide = padded(_randn(gen, total, scale=0.02))
    s = dict(case=c, step=40, flat=dict(p=wide.to(dt)), lists={})
    if c["master"]:
        s["flat"]["master"] = wide
    s["flat"]["grad"] = padded(_randn(gen, total, scale=1e-3)).to(dt)
    m = padded(_randn(gen, total, scale=3e-4))
    v = padded(_randn(gen, total, scale=1e-3).square_())
    if c["bits"] == 8:
        s["flat"]["m"], s["flat"]["m_scale"] = _encode(m, False)
        s["flat"]["v"], s["flat"]["v_scale"] = _encode(v.sqrt_(), True)
    else:
        s["flat"]["m"], s["flat"]["v"] = m, v
    for k, x in s["flat"].items():
        s["lists"][k] = views(x, BLOCK if k.endswith("_scale") else 1)
    # the clipping coefficient of the gradient's norm, left on the device
    s["grad_scale"] = torch.full((), 0.75, device=DEV)
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _first_rows(s, rows):
    """True at each sequence's first row, and the sequences that have one."""
    cu = s["cu"].long()
    full = (cu[1:] > cu[:-1]).nonzero().flatten()
    first = torch.zeros(rows, dtype=torch.bool, device=DEV)
    first[cu[full]] = True
    return first, full, cu


def _scan_rows(a, x, longest):
    """h_r = a_r h_{r-1} + x_r down the rows by doubling spans; overwrites both."""
    span = 1
    while span < longest:
        x[span:] += a[span:] * x[:-span]
        a[span:] = a[span:] * a[:-span]
        span *= 2
    return x


def _plain_scan(s):
    c = s["case"]
    shape, d = s["v"].shape, c["d"]
    rows = shape[0] * shape[1]
    flat = lambda x: x.detach().reshape(rows, d).float()  # noqa: E731
    v, a, h0 = flat(s["v"]), flat(s["g"]).exp(), s["h0"].detach()
    w = flat(s["w"]) if s["w"] is not None else None
    first, full, cu = _first_rows(s, rows)
    x = v * w if w is not None else v.clone()
    x[first] += a[first] * h0[full]
    kept = a.masked_fill(first[:, None], 0.0)
    h = _scan_rows(kept.clone(), x, s["longest"])
    ht = h0.clone()
    ht[full] = h[cu[full + 1] - 1]
    out = dict(y=h.view(shape).to(s["v"].dtype), ht=ht)
    if not c["train"]:
        return out
    last = cu[full + 1] - 1
    dy = flat(s["dy"])
    dy[last] += s["dht"][full]
    after = torch.zeros_like(a)
    after[:-1] = kept[1:]
    dh = _scan_rows(after.flip(0), dy.flip(0), s["longest"]).flip(0)
    before = torch.zeros_like(h)
    before[1:] = h[:-1]
    before[first] = h0[full]
    dh0 = s["dht"].clone()
    dh0[full] = a[first] * dh[first]
    like = lambda x, y: x.view(shape).to(y.dtype)  # noqa: E731
    out.update(dv=like(dh * w if w is not None else dh, s["v"]), dg=like(a * before * dh, s["g"]), dh0=dh0)
    if w is not None:
        out["dw"] = like(v * dh, s["w"])
    return out


def _plain_scan_step(s):
    at = s["slots"].long()
    x = s["v"].float()
    if s["w"] is not None:
        x = x * s["w"].float()
    h = s["g"].float().exp() * s["pool"][at] + x
    s["pool"][at] = h
    return dict(y=h.to(s["v"].dtype), pool=s["pool"])


def _top(z, k):
    """The ``k`` largest of each row, ties to the lowest index: one whole-number key for each value."""
    bits = (z + 0.0).view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    key = order * (1 << 32) + ((1 << 31) - 1 - torch.arange(z.shape[1], device=DEV))
    key = key.topk(k, dim=1).values
    at = (1 << 31) - 1 - (key & 0xFFFFFFFF)
    return z.gather(1, at), at


def _plain_logp(s):
    c = s["case"]
    z = s["logits"].detach().float() * (1.0 / c["temperature"])
    ids = s["ids"]
    on = ids != IGNORE
    at = ids.clamp(min=0)[:, None]
    low = z - z.amax(1, keepdim=True)
    e = low.exp()
    total = e.sum(1, keepdim=True)
    logp = low.gather(1, at) - total.log()
    out = dict(logp=torch.where(on, logp[:, 0], 0.0))
    p = e / total
    if c["entropy"]:
        finite = torch.where(e > 0, low, 0.0)
        ent = total.log() - (p * finite).sum(1, keepdim=True)
        out["entropy"] = torch.where(on, ent[:, 0], 0.0)
    if c["top"]:
        best, out["top_ids"] = _top(z, c["top"])
        out["top_logp"] = best - z.amax(1, keepdim=True) - total.log()
    if c["train"]:
        dl = (s["dlogp"] * on)[:, None]
        coef = -dl
        if c["entropy"]:
            coef = coef - (s["dent"] * on)[:, None] * (finite - total.log() + ent)
        dz = p * coef
        dz.scatter_add_(1, at, dl)
        out["dlogits"] = (dz * (1.0 / c["temperature"])).to(s["logits"].dtype)
    return out


def _encode(x, nonzero):
    """8-bit codes of a flat tensor and one scale for each block of it."""
    b = x.view(-1, BLOCK)
    most = b.abs().amax(1, keepdim=True)
    some = most > 1e-30
    inv = torch.where(some, 448.0 / most, 0.0)
    q = (b * inv).to(torch.float8_e4m3fn)
    if nonzero:  # a second moment that is not zero never becomes zero
        q = torch.where((b > 0) & some & (q.float() == 0), 2.0 ** -9, q.float()).to(torch.float8_e4m3fn)
    return q.view(-1), torch.where(some, most * (1.0 / 448.0), 0.0).view(-1)


def _decode(q, scale):
    return (q.float().view(-1, BLOCK) * scale[:, None]).view(-1)


def _plain_adamw(s):
    s["step"] += 1
    f, c = s["flat"], s["case"]
    b1, b2 = HYPER["beta1"], HYPER["beta2"]
    bc1, bc2 = 1 - b1 ** s["step"], 1 - b2 ** s["step"]
    g = f["grad"].float() * s["grad_scale"]
    p = f["master"] if c["master"] else f["p"].float()
    eight = c["bits"] == 8
    m = _decode(f["m"], f["m_scale"]) if eight else f["m"]
    v = _decode(f["v"], f["v_scale"]).square_() if eight else f["v"]
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    r = v.sqrt()
    p = p * (1 - HYPER["lr"] * HYPER["weight_decay"])
    p = p - (HYPER["lr"] / bc1) * m / (r * (1 / math.sqrt(bc2)) + HYPER["eps"])
    if eight:
        for k, x in (("m", m), ("v", r)):
            q, scale = _encode(x, k == "v")
            f[k].copy_(q)
            f[k + "_scale"].copy_(scale)
    else:
        f["m"].copy_(m)
        f["v"].copy_(v)
    if c["master"]:
        f["master"].copy_(p)
    f["p"].copy_(p)
    return {k: x for k, x in f.items() if k != "grad"}


# ---------------------------------------------------------------------------
# the framework's operators
# ---------------------------------------------------------------------------
def _own_scan(s):
    from qwendopamine_b200 import gated_scan

    c = s["case"]
    y, ht = gated_scan(s["v"], s["g"], s["w"], initial_state=s["h0"], output_final_state=True,
                       cu_seqlens=s["cu"] if c["seqs"] else None)
    out = dict(y=y.detach(), ht=ht.detach())
    if c["train"]:
        names = [k for k in ("v", "g", "w", "h0") if s[k] is not None]
        grads = torch.autograd.grad((y, ht), [s[k] for k in names], (s["dy"], s["dht"]))
        out.update(("d" + k, x) for k, x in zip(names, grads))
    return out


def _own_scan_step(s):
    from qwendopamine_b200 import gated_scan_step

    y = gated_scan_step(s["v"], s["g"], s["w"], state=s["pool"], state_indices=s["slots"])
    return dict(y=y, pool=s["pool"])


def _own_logp(s):
    from qwendopamine_b200 import token_logprobs

    c = s["case"]
    r = token_logprobs(s["logits"], s["ids"], top_k=c["top"], entropy=c["entropy"],
                       temperature=c["temperature"], ignore_index=IGNORE)
    out = dict(logp=r.logprobs.detach())
    if c["entropy"]:
        out["entropy"] = r.entropy.detach()
    if c["top"]:
        out["top_logp"], out["top_ids"] = r.top_logprobs, r.top_ids
    if c["train"]:
        ys, ds = (r.logprobs,), (s["dlogp"],)
        if c["entropy"]:
            ys, ds = (r.logprobs, r.entropy), (s["dlogp"], s["dent"])
        out["dlogits"], = torch.autograd.grad(ys, [s["logits"]], ds)
    return out


def _own_adamw(s):
    from qwendopamine_b200 import adamw_step

    s["step"] += 1
    t = s["lists"]
    adamw_step(t["p"], t["grad"], t["m"], t["v"], step=s["step"], lr=HYPER["lr"],
               betas=(HYPER["beta1"], HYPER["beta2"]), eps=HYPER["eps"],
               weight_decay=HYPER["weight_decay"], exp_avg_scales=t.get("m_scale"),
               exp_avg_sq_scales=t.get("v_scale"), master_params=t.get("master"),
               grad_scale=s["grad_scale"])
    return {k: x for k, x in s["flat"].items() if k != "grad"}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"scan": _own_scan, "scan_step": _own_scan_step, "logp": _own_logp,
                "adamw": _own_adamw}[op](state)
    with torch.no_grad():
        return {"scan": _plain_scan, "scan_step": _plain_scan_step, "logp": _plain_logp,
                "adamw": _plain_adamw}[op](state)


# ---------------------------------------------------------------------------
# work and exact values
# ---------------------------------------------------------------------------
def work(case):
    c = case
    e = SIZE[c["dtype"]]
    if c["op"] == "scan_step":
        n = c["n"] * c["d"]
        return dict(bytes=n * (2 * e + SIZE[c["gdtype"]] + e * c["gate"] + 8), flops=4 * n)
    if c["op"] == "scan":
        n, states = c["b"] * c["t"] * c["d"], (c["seqs"] or c["b"]) * c["d"]
        ins = e + SIZE[c["gdtype"]] + e * c["gate"]
        if c["train"]:
            return dict(bytes=n * (2 * ins + 2 * e) + 16 * states, flops=16 * n)
        return dict(bytes=n * (ins + e) + 8 * states, flops=4 * n)
    if c["op"] == "logp":
        n = c["rows"] * c["vocab"]
        return dict(bytes=n * e * (2 if c["train"] else 1) + c["rows"] * (12 + 12 * c["top"]),
                    flops=n * (4 + 2 * c["entropy"] + (5 if c["train"] else 0)))
    n = sum(_count(sh) for sh in _shapes(c))
    state = 4 + 16 / BLOCK if c["bits"] == 8 else 16
    return dict(bytes=n * ((e + 8 + e if c["master"] else 2 * e + e) + state), flops=16 * n)


def _exact_scan(s):
    """Row by row from the definition."""
    c = s["case"]
    rows = s["v"].shape[0] * s["v"].shape[1]
    wide = lambda x: x.detach().double().reshape(rows, c["d"])  # noqa: E731
    v, a = wide(s["v"]), wide(s["g"]).exp()
    w = wide(s["w"]) if s["w"] is not None else torch.ones_like(v)
    h0 = s["h0"].detach().double()
    if c["seqs"]:
        spans = [(n, lo, hi) for n, (lo, hi) in enumerate(zip(s["cu"].tolist(), s["cu"].tolist()[1:]))]
        pick = lambda x: [x[lo:hi] for _, lo, hi in spans]  # noqa: E731
    else:
        pick = lambda x: [x.view(c["b"], c["t"], c["d"]).transpose(0, 1)]  # noqa: E731
        spans = [(slice(None), 0, c["t"])]
    x = w * v
    y, ht, prev = torch.empty_like(v), h0.clone(), torch.empty_like(v)
    for (n, lo, hi), av, xv, yv, pv in zip(spans, pick(a), pick(x), pick(y), pick(prev)):
        h = h0[n]
        for t in range(hi - lo):
            pv[t] = h
            h = torch.addcmul(xv[t], av[t], h)
            yv[t] = h
        ht[n] = h
    out = dict(y=y.view(s["v"].shape), ht=ht)
    if c["train"]:
        dy, dht = wide(s["dy"]), s["dht"].double()
        dh, dh0 = torch.empty_like(v), dht.clone()
        for (n, lo, hi), av, dv, ov in zip(spans, pick(a), pick(dy), pick(dh)):
            carry = dht[n]
            for t in range(hi - lo - 1, -1, -1):
                z = dv[t] + carry
                ov[t] = z
                carry = av[t] * z
            dh0[n] = carry
        shaped = lambda z: z.view(s["v"].shape)  # noqa: E731
        out.update(dv=shaped(w * dh), dg=shaped(a * prev * dh), dh0=dh0)
        if s["w"] is not None:
            out["dw"] = shaped(v * dh)
    return out


def _exact_logp(s):
    """A few rows at a time, through log_softmax in 64 bits and a stable sort."""
    c = s["case"]
    names = ["logp"] + ["entropy"] * c["entropy"] + ["top_logp", "top_ids"] * (c["top"] > 0)
    names += ["dlogits"] * c["train"]
    parts = {k: [] for k in names}
    for lo in range(0, c["rows"], 64):
        z = s["logits"].detach()[lo: lo + 64].double() / c["temperature"]
        ids = s["ids"][lo: lo + 64]
        on = (ids != IGNORE).double()
        lp = torch.log_softmax(z, 1)
        p = lp.exp()
        finite = lp.masked_fill(p == 0, 0.0)
        hot = torch.zeros_like(z)
        hot[torch.arange(len(ids), device=DEV), ids.clamp(min=0)] = 1.0
        parts["logp"].append((finite * hot).sum(1) * on)
        ent = -(p * finite).sum(1)
        if c["entropy"]:
            parts["entropy"].append(ent * on)
        if c["top"]:
            order = torch.sort(z, dim=1, descending=True, stable=True).indices[:, : c["top"]]
            parts["top_ids"].append(order)
            parts["top_logp"].append(lp.gather(1, order))
        if c["train"]:
            dl = s["dlogp"][lo: lo + 64].double() * on
            d = dl[:, None] * (hot - p)
            if c["entropy"]:
                de = s["dent"][lo: lo + 64].double() * on
                d = d - de[:, None] * p * (finite + ent[:, None])
            parts["dlogits"].append(d / c["temperature"])
    return {k: torch.cat(x) for k, x in parts.items()}


def _exact_adamw(s):
    f, c = s["flat"], s["case"]
    t = s["step"] + 1
    b1, b2 = HYPER["beta1"], HYPER["beta2"]
    g = f["grad"].double() * float(s["grad_scale"])
    p = f["master" if c["master"] else "p"].double()
    if c["bits"] == 8:
        m = f["m"].double() * f["m_scale"].double().repeat_interleave(BLOCK)
        v = (f["v"].double() * f["v_scale"].double().repeat_interleave(BLOCK)) ** 2
    else:
        m, v = f["m"].double(), f["v"].double()
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g ** 2
    mhat, vhat = m / (1 - b1 ** t), v / (1 - b2 ** t)
    p = p - HYPER["lr"] * (mhat / (vhat.sqrt() + HYPER["eps"]) + HYPER["weight_decay"] * p)
    out = dict(p=p, m=m, v=v)
    if c["master"]:
        out["master"] = p
    if c["bits"] == 8:
        for k, x in (("m", m), ("v", v.sqrt())):
            b = x.view(-1, BLOCK)
            most = b.abs().amax(1, keepdim=True)
            u = torch.where(most > 0, b / most * 448, 0.0)
            step = 2.0 ** (torch.floor(torch.log2(u.abs().clamp(min=2.0 ** -6))) - 3)
            q = torch.round(u / step) * step
            if k == "v":
                q = torch.where((u > 0) & (q == 0), 2.0 ** -9, q)
            out[k], out[k + "_scale"] = q.view(-1), (most / 448).view(-1)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "scan":
        return _exact_scan(s)
    if case["op"] == "logp":
        return _exact_logp(s)
    if case["op"] == "adamw":
        return _exact_adamw(s)
    at = s["slots"].long()
    w = s["w"].double() if s["w"] is not None else 1.0
    h = s["g"].double().exp() * s["pool"][at].double() + w * s["v"].double()
    pool = s["pool"].double()
    pool[at] = h
    return dict(y=h, pool=pool)
