"""AdamW on the GPU against the float64 oracle.

Tolerances.  fp32 results are a handful of fp32 operations on exact inputs: a
state element's relative error stays below 4 * 2^-24 plus cancellation in
m = b1 m + (1-b1) g; relative L2 1e-6.  The change of a parameter, lr-sized,
is compared through the parameter itself: 1e-6 for fp32; 16-bit parameters add
one rounding of at most 2^-9 / 2^-12, doubled.  8-bit states: a code may differ
from the oracle's where fp32 and fp64 fall on two sides of a rounding
boundary: at most one code in a thousand, by one step of at most 1/8.
"""

import numpy as np
import pytest
import torch

from oracle import op_oracle as O
from qwendopamine_b200 import AdamW, adamw_step

pytestmark = pytest.mark.gpu

F32, BF, FH = torch.float32, torch.bfloat16, torch.float16
F8 = torch.float8_e4m3fn
TOL = {F32: 1e-6, BF: 2.0 ** -8, FH: 2.0 ** -11}
H = dict(lr=3e-3, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)
SIZES = [1, 7, 8, 255, 256, 257, 8191, 8192, 8193, 0, 100003]


def np64(t):
    return t.detach().double().cpu().numpy().ravel()


def close(got, want, dtype=None):
    a = np64(got)
    assert np.isfinite(a).all()
    err = np.linalg.norm(a - want) / max(np.linalg.norm(want), 1e-30)
    assert err <= TOL[dtype or got.dtype], err


def make(dev, dtype, gdtype, bits, master, sizes=SIZES, seed=0, offset=0):
    """Lists of tensors, `offset` elements into their storage."""
    gen = torch.Generator().manual_seed(seed)

    def new(x, dt):
        buf = torch.zeros(x.numel() + offset, device=dev).to(dt)
        buf[offset:] = x.to(dev, dt) if dt != F8 else x.to(dev)
        return buf[offset:]

    rn = lambda n, s: torch.randn(n, generator=gen) * s
    out = {k: [] for k in ("p", "g", "m", "v", "ms", "vs", "w")}
    for n in sizes:
        w = rn(n, 0.02)
        out["p"].append(new(w, dtype))
        out["w"].append(new(w, F32))
        out["g"].append(new(rn(n, 1e-2), gdtype))
        m, v = rn(n, 3e-3), rn(n, 1e-2) ** 2
        if bits == 32:
            out["m"].append(new(m, F32))
            out["v"].append(new(v, F32))
            continue
        for k, x in (("m", m), ("v", v.sqrt())):
            codes, scales = O.encode8(x.double().numpy(), k == "v")
            buf = torch.zeros(n + offset, dtype=torch.uint8, device=dev).view(F8)
            buf[offset:] = torch.from_numpy(codes).float().to(F8).to(dev)
            out[k].append(buf[offset:])
            out[k + "s"].append(torch.from_numpy(scales).float().to(dev))
    return out


def call(x, bits, master, step=7, **kw):
    adamw_step(x["p"], x["g"], x["m"], x["v"], step=step, **{**H, **kw},
               exp_avg_scales=x["ms"] if bits == 8 else None,
               exp_avg_sq_scales=x["vs"] if bits == 8 else None,
               master_params=x["w"] if master else None)


def values8(codes, scales):
    return np64(codes) * np.repeat(np64(scales), 256)[:codes.numel()]


def expected(x, i, bits, master, step=7, scale=1.0, lr=H["lr"]):
    p = np64(x["w" if master else "p"][i])
    if bits == 8:
        m, v = values8(x["m"][i], x["ms"][i]), values8(x["v"][i], x["vs"][i]) ** 2
    else:
        m, v = np64(x["m"][i]), np64(x["v"][i])
    return O.adamw(p, np64(x["g"][i]) * scale, m, v, step, lr, *H["betas"], H["eps"],
                   H["weight_decay"])


def check_state(got, scales, want, nonzero):
    codes, sc = O.encode8(want, nonzero)
    assert np.allclose(np64(scales), sc, rtol=1e-6, atol=0)
    a = np64(got)
    off = a != codes
    assert off.mean() <= 1e-3
    assert (np.abs(a - codes)[off] <= np.maximum(np.abs(codes[off]) / 8, 2.0 ** -9)).all()


def check(x, bits, master, **kw):
    scale = kw.pop("scale", 1.0)
    want = [expected(x, i, bits, master, scale=scale) for i in range(len(x["p"]))]
    if scale != 1.0:
        kw["grad_scale"] = torch.tensor(scale, device=x["p"][0].device)
    call(x, bits, master, **kw)
    for i, (p, m, v) in enumerate(want):
        if p.size == 0:
            continue
        close(x["p"][i], p)
        if master:
            close(x["w"][i], p)
        if bits == 32:
            close(x["m"][i], m)
            close(x["v"][i], v)
        else:
            check_state(x["m"][i], x["ms"][i], m, False)
            check_state(x["v"][i], x["vs"][i], np.sqrt(v), True)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("master", [False, True])
@pytest.mark.parametrize("dtype,gdtype", [(F32, F32), (BF, BF), (BF, F32), (FH, FH), (FH, F32)])
def test_sizes_and_types(cuda_device, dtype, gdtype, master, bits):
    check(make(cuda_device, dtype, gdtype, bits, master), bits, master)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("offset", [1, 4])
def test_storage_offsets(cuda_device, offset, bits):
    check(make(cuda_device, BF, BF, bits, True, offset=offset, seed=1), bits, True)


@pytest.mark.parametrize("bits", [32, 8])
def test_more_tensors_than_one_launch_takes(cuda_device, bits):
    x = make(cuda_device, BF, BF, bits, False, sizes=[5 + i % 300 for i in range(901)], seed=2)
    check(x, bits, False)


@pytest.mark.parametrize("bits", [32, 8])
def test_gradient_scale_and_found_inf(cuda_device, bits):
    x = make(cuda_device, F32, F32, bits, False, seed=3)
    check(x, bits, False, scale=0.25)
    keep = {k: [t.clone() for t in v] for k, v in x.items()}
    one, zero = torch.ones((), device=cuda_device), torch.zeros((), device=cuda_device)
    x["g"][-1][5] = float("inf")
    call(x, bits, False, found_inf=one)
    for k in ("p", "m", "v", "ms", "vs"):
        for a, b in zip(keep[k], x[k]):
            assert torch.equal(a.view(torch.uint8) if a.dtype == F8 else a,
                               b.view(torch.uint8) if b.dtype == F8 else b)
    x["g"][-1][5] = 0
    call(x, bits, False, found_inf=zero)
    assert not torch.equal(keep["p"][-1], x["p"][-1])


def test_8bit_codes_at_their_limits(cuda_device):
    """Blocks of zeros, of one huge and many tiny values, and below 1e-30; a
    small second moment does not become zero."""
    n = 256 * 5
    x = make(cuda_device, F32, F32, 8, False, sizes=[n], seed=4)
    for k in ("m", "v"):
        x[k][0].view(torch.uint8).zero_()
        x[k + "s"][0].zero_()
    g = torch.zeros(n)
    g[256:512] = 1e-6
    g[300] = 1e3
    g[512:768] = torch.randn(256) * 1e-32
    g[768:] = torch.logspace(-12, 3, 512)
    x["g"][0].copy_(g)
    p, m, v = expected(x, 0, 8, False, step=1)
    call(x, 8, False, step=1)
    check_state(x["m"][0], x["ms"][0], m, False)
    # the root of v in fp32: squares below 2^-149 are zero
    v32 = np.where(v < 2.0 ** -149, 0, v)
    r = np64(x["v"][0])
    assert (r[v32 > 0][np.sqrt(v32[v32 > 0]) > 1e-20] > 0).all()
    assert (r[:256] == 0).all() and (r[512:768] == 0).all()
    assert r[256] == 2.0 ** -9 and r[300] == 448
    for _ in range(3):
        call(x, 8, False, step=2)
    assert x["p"][0].isfinite().all() and x["p"][0].abs().max() < 1


@pytest.mark.parametrize("bits", [32, 8])
def test_gradients_whose_squares_overflow(cuda_device, bits):
    """A gradient of 1e30 moves its parameter by a step's size at most and
    leaves its neighbours alone; a NaN stays where it is."""
    x = make(cuda_device, F32, F32, bits, False, sizes=[256, 512], seed=10)
    x["g"][0][7] = 1e30
    x["g"][1][300] = float("nan")
    before = [p.clone() for p in x["p"]]
    call(x, bits, False, step=1, weight_decay=0.0)
    assert x["p"][0].isfinite().all()
    assert (x["p"][0] - before[0])[7].abs() <= 2 * H["lr"] / (1 - H["betas"][0])
    bad = x["p"][1].isnan()
    assert bad[300] and int(bad.sum()) == 1


def test_many_steps_with_8bit_states_follow_32bit(cuda_device):
    """A least-squares problem: both reach the same loss."""
    gen = torch.Generator().manual_seed(5)
    A = torch.randn(512, 64, generator=gen).to(cuda_device)
    y = A @ torch.randn(64, 33, generator=gen).to(cuda_device)
    losses = []
    for bits in (32, 8):
        w = torch.nn.Parameter(torch.zeros(64, 33, device=cuda_device))
        opt = AdamW([w], lr=0.05, weight_decay=0.0, state_bits=bits)
        for _ in range(300):
            opt.zero_grad()
            loss = (A @ w - y).square().mean()
            loss.backward()
            opt.step()
        losses.append(float(loss))
    start = float(y.square().mean())
    assert losses[0] < 1e-3 * start and losses[1] < 1e-2 * start


@pytest.mark.parametrize("bits,master", [(32, False), (8, False), (8, True), (32, True)])
def test_optimizer_resumes_from_its_state_dict(cuda_device, bits, master):
    gen = torch.Generator().manual_seed(6)
    init = [torch.randn(37, 11, generator=gen), torch.randn(300, generator=gen)]
    grads = [[torch.randn(p.shape, generator=gen) for p in init] for _ in range(6)]

    def fresh():
        ps = [torch.nn.Parameter(p.to(cuda_device, BF)) for p in init]
        return ps, AdamW([{"params": ps[:1]}, {"params": ps[1:], "weight_decay": 0.0}], lr=1e-2,
                         state_bits=bits, master_weights=master)

    def run(ps, opt, part):
        for gs in part:
            for p, g in zip(ps, gs):
                p.grad = g.to(cuda_device, BF)
            opt.step()

    ps, opt = fresh()
    run(ps, opt, grads)
    qs, first = fresh()
    run(qs, first, grads[:3])
    saved = first.state_dict()
    rs, second = fresh()
    for r, q in zip(rs, qs):
        r.data.copy_(q)
    second.load_state_dict(saved)
    run(rs, second, grads[3:])
    for a, b in zip(ps, rs):
        assert torch.equal(a, b)
    for a, b in zip(ps, rs):
        for k, t in opt.state[a].items():
            u = second.state[b][k]
            if isinstance(t, torch.Tensor):
                assert t.dtype == u.dtype
                assert torch.equal(t.view(torch.uint8) if t.dtype == F8 else t,
                                   u.view(torch.uint8) if u.dtype == F8 else u)
            else:
                assert t == u


def test_optimizer_matches_the_oracle_over_steps(cuda_device):
    gen = torch.Generator().manual_seed(7)
    w = torch.randn(70, 9, generator=gen)
    p = torch.nn.Parameter(w.to(cuda_device))
    idle = torch.nn.Parameter(torch.ones(4, device=cuda_device))
    opt = AdamW([p, idle], **H)
    ref = (w.double().numpy().ravel(), np.zeros(630), np.zeros(630))
    for t in range(1, 9):
        g = torch.randn(9, 70, generator=gen).t()  # not contiguous
        p.grad = g.to(cuda_device)
        ref = O.adamw(ref[0], g.double().numpy().ravel(), *ref[1:], t, H["lr"], *H["betas"],
                      H["eps"], H["weight_decay"])
        assert opt.step(closure=lambda: 3.0) == 3.0
    close(p, ref[0])
    assert idle.eq(1).all() and not opt.state[idle]


def test_a_tensor_beyond_32_bits(cuda_device):
    n = (1 << 31) + 1029
    p = torch.zeros(n, dtype=BF, device=cuda_device)
    g = torch.zeros(n, dtype=BF, device=cuda_device)
    m = torch.zeros(n, dtype=torch.uint8, device=cuda_device).view(F8)
    v = torch.zeros(n, dtype=torch.uint8, device=cuda_device).view(F8)
    ms, vs = (torch.zeros(-(-n // 256), device=cuda_device) for _ in range(2))
    g[-1] = g[3] = g[(1 << 31) + 2] = 1.0
    adamw_step([p], [g], [m], [v], step=1, lr=0.5, weight_decay=0.0, exp_avg_scales=[ms],
               exp_avg_sq_scales=[vs])
    assert p[-1] == -0.5 and p[3] == -0.5 and p[(1 << 31) + 2] == -0.5
    assert int((p != 0).sum()) == 3
    assert float(m[-1].float() * ms[-1]) == pytest.approx(0.1, rel=1e-6)


def test_equal_inputs_give_equal_bits(cuda_device):
    runs = []
    for _ in range(2):
        x = make(cuda_device, BF, BF, 8, False, seed=8)
        for t in range(1, 5):
            call(x, 8, False, step=t)
        runs.append(x)
    for k in ("p", "m", "v", "ms", "vs"):
        for a, b in zip(runs[0][k], runs[1][k]):
            assert torch.equal(a.view(torch.uint8) if a.dtype == F8 else a,
                               b.view(torch.uint8) if b.dtype == F8 else b)


def test_refusals(cuda_device):
    new = lambda: make(cuda_device, BF, BF, 8, True, sizes=[300, 20], seed=9)

    def bad(match, exc=ValueError, bits=8, master=True, **kw):
        x = new()
        for k in list(kw):
            if k in x:
                x[k] = kw.pop(k)
        with pytest.raises(exc, match=match):
            call(x, bits, master, **kw)

    z = lambda n, dt=F32: torch.zeros(n, device=cuda_device, dtype=dt)
    bad("grads has 1", g=[z(300, BF)])
    bad("sizes", g=[z(300, BF), z(21, BF)])
    bad("must all be", m=[z(300), z(20)])
    bad("must all be", w=[z(300, BF), z(20, BF)])
    bad("one value for each", ms=[z(1), z(1)])
    bad("CUDA", RuntimeError, p=[torch.zeros(300, dtype=BF), torch.zeros(20, dtype=BF)])
    bad("float32 or have", NotImplementedError, g=[z(300, FH), z(20, FH)])
    bad("contiguous", p=[z(600, BF)[::2], z(20, BF)])
    bad("step", step=0)
    bad("betas", betas=(1.0, 0.9))
    bad("finite", lr=float("nan"))
    bad("grad_scale", grad_scale=torch.ones(2, device=cuda_device))
    x = new()
    with pytest.raises(ValueError, match="both"):
        adamw_step(x["p"], x["g"], x["m"], x["v"], step=1, **H, exp_avg_scales=x["ms"])
    with pytest.raises(ValueError, match="must all be"):
        call(x, 32, True)
    adamw_step([], [], [], [], step=1, **H)
    for kw in (dict(state_bits=16), dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(eps=-1.0)):
        with pytest.raises(ValueError):
            AdamW([torch.nn.Parameter(z(3))], **kw)
