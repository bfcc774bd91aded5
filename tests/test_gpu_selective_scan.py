"""Selective state space scan on the GPU against the float64 oracle.

Tolerances (relative L2).  fp32: a step rounds the decay's exponent (2^-24 of
A log2(e), 2^-24 of the product, times an exponent below 4) and takes the
hardware's base-2 exponential (2^-22), then two products and a sum: below 2^-20.5
in all, over an effective window of at most 30 steps at these decays (0.1 and more
in the exponent): 2e-5.  16-bit results: one rounding of a value that is right to
fp32, at most 2^-8 (bf16) or 2^-11 (fp16) of each element and 0.58 of that in the
mean over elements; the terms of dB and dC in bf16 have two factors rounded within
1.28 * 2^-11, a third of 2^-8 together.  States and
the gradients of fp32 inputs are fp32 results whatever the token type; so are dA,
dD, ddt_bias, whose terms with 16-bit gates carry 2^-21 more.
"""

import numpy as np
import pytest
import torch

from oracle import op_oracle as O
from qwendopamine_b200 import selective_scan, selective_scan_step

pytestmark = pytest.mark.gpu

TOL = {torch.float32: 2e-5, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
F32, BF, FH = torch.float32, torch.bfloat16, torch.float16
NAMES = ("x", "dt", "A", "B", "C", "D", "z", "dt_bias", "h0")


def np64(t):
    return None if t is None else t.detach().double().cpu().numpy()


def close(got, want, name="", dtype=None):
    a = np64(got)
    assert a.shape == want.shape, name
    assert np.isfinite(a).all(), name
    err = np.linalg.norm(a - want) / max(np.linalg.norm(want), 1e-30)
    assert err <= TOL[dtype or got.dtype], (name, err)


def inputs(dev, B, T, d, n, dtype, dtdtype, n_seqs, groups=None, gate=True, more=True, plus=True, seed=0):
    gen = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen)
    vec = (B, T, n) if groups is None else (B, T, groups, n)
    dt = rn(B, T, d) * 0.5 if plus else torch.rand(B, T, d, generator=gen) + 0.2
    v = dict(x=rn(B, T, d).to(dtype), dt=dt.to(dtdtype), A=-(0.5 + torch.rand(d, n, generator=gen)),
             B=rn(*vec).to(dtype), C=rn(*vec).to(dtype), D=rn(d) if more else None,
             z=rn(B, T, d).to(dtype) if gate else None, dt_bias=rn(d) * 0.1 if more else None,
             h0=rn(n_seqs, d, n), dy=rn(B, T, d).to(dtype), dht=rn(n_seqs, d, n))
    return {k: None if t is None else t.to(dev) for k, t in v.items()}


def run(v, plus=True, cu=None, use_h0=True):
    cut = None if cu is None else torch.tensor(cu, dtype=torch.int32, device=v["x"].device)
    return selective_scan(v["x"], v["dt"], v["A"], v["B"], v["C"], v["D"], v["z"], dt_bias=v["dt_bias"],
                          dt_softplus=plus, initial_state=v["h0"] if use_h0 else None,
                          output_final_state=True, cu_seqlens=cut)


def check(v, plus=True, cu=None, use_h0=True, use_dht=True, grads=True):
    args = [np64(v[k]) for k in NAMES[:8]] + [plus, np64(v["h0"]) if use_h0 else None]
    ry, _, rh = O.selective_fwd(*args, cu)
    with torch.no_grad():
        y0, h0 = run(v, plus, cu, use_h0)
    close(y0, ry, "y")
    close(h0, rh, "ht")
    if not grads:
        return
    leaves = {k: t.detach().requires_grad_() for k, t in v.items()
              if k in NAMES and t is not None and (k != "h0" or use_h0)}
    y, ht = run({**v, **leaves}, plus, cu, use_h0)
    assert torch.equal(y, y0) and torch.equal(ht, h0)
    outs, gout = ([y, ht], [v["dy"], v["dht"]]) if use_dht else ([y], [v["dy"]])
    got = dict(zip(leaves, torch.autograd.grad(outs, list(leaves.values()), gout)))
    want = O.selective_bwd(*args, np64(v["dy"]), np64(v["dht"]) if use_dht else None, cu)
    for k, g in got.items():
        assert g.dtype == v[k].dtype and g.shape == v[k].shape
        close(g, want[k], "d" + k)
    return got


TYPES = [(F32, F32), (BF, BF), (BF, F32), (FH, FH)]


@pytest.mark.parametrize("dtype,dtdtype", TYPES)
@pytest.mark.parametrize("B,T,d,n", [(1, 1, 1, 1), (3, 1, 40, 16), (2, 5, 7, 3), (1, 15, 33, 16), (2, 16, 32, 8),
                                     (2, 17, 64, 16), (1, 33, 70, 13), (2, 50, 20, 32), (1, 40, 9, 64),
                                     (1, 20, 17, 41)])
def test_fixed_length(cuda_device, B, T, d, n, dtype, dtdtype):
    check(inputs(cuda_device, B, T, d, n, dtype, dtdtype, B))


@pytest.mark.parametrize("T,d,n", [(64, 8, 16), (65, 40, 16), (1000, 40, 16), (777, 70, 8), (500, 24, 40)])
def test_time_axis_cut_into_chunks(cuda_device, T, d, n):
    check(inputs(cuda_device, 2, T, d, n, F32, F32, 2, seed=1))


def test_one_chunk_where_channels_fill_the_gpu(cuda_device):
    check(inputs(cuda_device, 300, 70, 33, 4, BF, F32, 300, seed=2))


@pytest.mark.parametrize("dtype,dtdtype", TYPES)
@pytest.mark.parametrize("n", [4, 16])
def test_packed_sequences(cuda_device, n, dtype, dtdtype):
    lens = [0, 1, 5, 0, 0, 15, 16, 17, 1, 300, 64, 0, 128, 2, 0]
    cu = np.concatenate([[0], np.cumsum(lens)]).tolist()
    check(inputs(cuda_device, 1, cu[-1], 36, n, dtype, dtdtype, len(lens), seed=3), cu=cu)


def test_many_short_sequences_and_one_long(cuda_device):
    check(inputs(cuda_device, 1, 200, 20, 16, F32, F32, 200, seed=4), cu=list(range(201)))
    check(inputs(cuda_device, 1, 700, 20, 16, F32, F32, 1, seed=4), cu=[0, 700])


@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("more", [False, True])
@pytest.mark.parametrize("plus", [False, True])
def test_without_options(cuda_device, gate, more, plus):
    v = inputs(cuda_device, 2, 70, 24, 16, F32, F32, 2, gate=gate, more=more, plus=plus, seed=5)
    check(v, plus)
    check(v, plus, use_h0=False)
    check(v, plus, use_dht=False)


@pytest.mark.parametrize("groups,d", [(1, 40), (2, 40), (5, 40), (3, 300), (40, 40)])
@pytest.mark.parametrize("n", [16, 6])
def test_groups_of_channels(cuda_device, groups, d, n):
    check(inputs(cuda_device, 2, 37, d, n, BF, F32, 2, groups=groups, seed=6))


def test_gradient_of_the_end_state_alone(cuda_device):
    v = inputs(cuda_device, 2, 90, 12, 16, F32, F32, 2, seed=7)
    leaves = [v[k].requires_grad_() for k in NAMES]
    _, ht = run(v)
    got = torch.autograd.grad(ht, leaves, v["dht"])
    want = O.selective_bwd(*(np64(v[k]) for k in NAMES[:8]), True, np64(v["h0"]), np.zeros((2, 90, 12)),
                           np64(v["dht"]))
    for k, g in zip(NAMES, got):
        if k in ("C", "z", "D"):
            assert not g.any()
        else:
            close(g, want[k], k)


def test_extreme_decays(cuda_device):
    """A product of decays that underflows, no decay at all, and slow growth."""
    for lo, hi in ((-300.0, -100.0), (0.0, 0.0), (0.0, 0.002)):
        v = inputs(cuda_device, 2, 200, 16, 16, F32, F32, 2, seed=8)
        v["A"] = (torch.rand(16, 16, generator=torch.Generator().manual_seed(9)) * (hi - lo) + lo).to(cuda_device)
        if lo == 0.0:
            # 200 steps without decay: the window is the whole sequence, 200 * 2^-22
            v["x"] = v["x"].abs()
        check(v) if lo < 0 else check_loose(v, 200 * 2.0 ** -21)


def check_loose(v, tol):
    keep = TOL[F32]
    TOL[F32] = tol
    try:
        check(v)
    finally:
        TOL[F32] = keep


def test_small_steps_keep_their_softplus(cuda_device):
    """softplus of very negative numbers is their exponential, not zero."""
    v = inputs(cuda_device, 1, 100, 16, 16, F32, F32, 1, seed=10)
    v["dt"] = v["dt"] - 14.0
    # decays of 1 - 1e-6: a window of the 100 steps, 100 * 2^-21
    check_loose(v, 100 * 2.0 ** -21)


def test_strided_rows(cuda_device):
    """Slices of fused projections: x and z of one, dt, B and C of another."""
    v = inputs(cuda_device, 2, 40, 24, 16, BF, BF, 2, seed=11)
    a = torch.cat([v["x"], v["z"], v["dy"]], -1)
    b = torch.cat([v["dt"], v["B"], v["C"]], -1)
    v["x"], v["z"], v["dy"] = a.split([24, 24, 24], -1)
    v["dt"], v["B"], v["C"] = b.split([24, 16, 16], -1)
    assert not v["x"].is_contiguous() and not v["C"].is_contiguous()
    check(v)
    v["x"] = v["x"].transpose(0, 1).contiguous().transpose(0, 1)
    v["B"] = v["B"].transpose(1, 2).contiguous().transpose(1, 2)
    check(v)


def test_parameters_in_16_bits(cuda_device):
    v = inputs(cuda_device, 2, 40, 24, 16, BF, BF, 2, seed=12)
    for k in ("A", "D", "dt_bias"):
        v[k] = v[k].to(BF)
    check(v)


def test_empty_batches_and_sequences(cuda_device):
    v = inputs(cuda_device, 1, 4, 8, 16, F32, F32, 3, seed=13)
    none = {k: t[:, :0] for k, t in v.items() if k in ("x", "dt", "B", "C", "z")}
    y, ht = run({**v, **none}, cu=[0, 0, 0, 0])
    assert y.shape == (1, 0, 8) and torch.equal(ht, v["h0"])
    h0 = v["h0"][:1].clone().requires_grad_()
    A = v["A"].clone().requires_grad_()
    y, ht = run({**v, **none, "h0": h0, "A": A})
    dA, dh = torch.autograd.grad(ht, [A, h0], v["dht"][:1])
    assert torch.equal(dh, v["dht"][:1]) and not dA.any()
    y, ht = selective_scan(*(v[k][:0] if k in ("x", "dt", "B", "C") else v[k] for k in ("x", "dt", "A", "B", "C")),
                           output_final_state=True)
    assert y.shape == (0, 4, 8) and ht.shape == (0, 8, 16)


def test_a_sequence_does_not_see_its_neighbours_nan(cuda_device):
    cu = [0, 20, 37, 60]
    v = inputs(cuda_device, 1, 60, 12, 16, F32, F32, 3, seed=14)
    leaves = {k: v[k].requires_grad_() for k in ("x", "B", "h0")}
    y, ht = run({**v, **leaves}, cu=cu)
    clean = (y, ht, *torch.autograd.grad((y, ht), list(leaves.values()), (v["dy"], v["dht"])))
    with torch.no_grad():
        v["x"][:, 25] = torch.nan
        v["dy"][:, 30] = torch.inf
    y, ht = run({**v, **leaves}, cu=cu)
    dirty = (y, ht, *torch.autograd.grad((y, ht), list(leaves.values()), (v["dy"], v["dht"])))
    for c, d, seqs in zip(clean, dirty, (False, True, False, False, True)):
        if seqs:
            assert torch.equal(c[[0, 2]], d[[0, 2]])
        else:
            assert torch.equal(c[:, :20], d[:, :20]) and torch.equal(c[:, 37:], d[:, 37:])


@pytest.mark.parametrize("dtype", [F32, BF, FH])
@pytest.mark.parametrize("n", [4, 16, 40])
def test_nan_reaches_what_it_is_in(cuda_device, n, dtype):
    """A NaN in x is in y, dC and dA from its row on, in dB in its row alone; one in
    dy is in dB and dx up to its row."""
    for name, row in (("x", 25), ("dy", 40)):
        v = inputs(cuda_device, 1, 70, 12, n, dtype, dtype, 1, seed=24)
        v[name][:, row] = torch.nan
        leaves = [v[k].requires_grad_() for k in ("x", "A", "B", "C")]
        y, _ = run(v)
        dx, dA, dB, dC = torch.autograd.grad(y, leaves, v["dy"])
        at = torch.arange(70, device=cuda_device)[None, :, None]
        nan = lambda t, rows: torch.equal(t.isnan(), rows.expand(t.shape))
        assert dA.isnan().all()
        if name == "x":
            assert nan(y, at >= row) and nan(dC, at >= row) and nan(dB, at == row) and not dx.isnan().any()
        else:
            assert not y.isnan().any() and nan(dC, at == row) and nan(dB, at <= row) and nan(dx, at <= row)


def test_equal_inputs_give_equal_bits(cuda_device):
    v = inputs(cuda_device, 1, 3000, 100, 16, BF, BF, 1, seed=15)
    a, b = check(v), check(v)
    assert all(torch.equal(a[k], b[k]) for k in a)


def test_scan_in_pieces_equals_the_whole(cuda_device):
    v = inputs(cuda_device, 1, 100, 32, 16, F32, F32, 1, seed=16)
    with torch.no_grad():
        y, ht = run(v)
        cut = lambda lo, hi: {k: t[:, lo:hi] if k in ("x", "dt", "B", "C", "z") else t for k, t in v.items()}
        y1, h1 = run(cut(0, 41))
        y2, h2 = run({**cut(41, 100), "h0": h1})
    close(torch.cat([y1, y2], 1), np64(y))
    close(h2, np64(ht))


@pytest.mark.parametrize("dtype,dtdtype", TYPES)
@pytest.mark.parametrize("n,d,states,groups", [(1, 1, 1, None), (5, 70, 16, None), (64, 48, 16, 2), (3, 33, 8, 3),
                                               (2, 20, 64, None), (4, 20, 13, 4), (601, 260, 16, None), (7, 33, 16, None),
                                               (299, 500, 6, 5)])
def test_step(cuda_device, n, d, states, groups, dtype, dtdtype):
    v = inputs(cuda_device, n, 1, d, states, dtype, dtdtype, n, groups=groups, seed=17)
    pool = torch.randn(n + 3, d, states, device=cuda_device)
    slots = torch.randperm(n + 3, device=cuda_device)[:n]
    before = pool.clone()
    one = {k: t[:, 0] if k in ("x", "dt", "B", "C", "z") and t is not None else t for k, t in v.items()}
    call = lambda st, idx: selective_scan_step(
        one["x"], one["dt"], one["A"], one["B"], one["C"], one["D"], one["z"], dt_bias=one["dt_bias"],
        dt_softplus=True, state=st, state_indices=idx)
    y = call(pool, slots)
    ry, _, rh = O.selective_fwd(*(np64(v[k]) for k in NAMES[:8]), True, np64(before[slots]))
    close(y, ry[:, 0])
    close(pool[slots], rh)
    rest = torch.ones(n + 3, dtype=torch.bool, device=cuda_device)
    rest[slots] = False
    assert torch.equal(pool[rest], before[rest])
    # without indices, and with rows of a wider pool
    wide = torch.randn(n, d * states + 5, device=cuda_device)
    view = wide[:, : d * states].view(n, d, states) if n > 1 else wide[:, : d * states].reshape(n, d, states)
    view.copy_(before[slots])
    tail = wide[:, d * states:].clone()
    assert torch.equal(call(view, None), y) and torch.equal(view, pool[slots])
    assert torch.equal(wide[:, d * states:], tail)


def test_step_padding_and_version(cuda_device):
    v = inputs(cuda_device, 4, 1, 20, 16, BF, F32, 4, seed=18)
    pool = torch.randn(3, 20, 16, device=cuda_device)
    before, version = pool.clone(), pool._version
    args = [v[k][:, 0] for k in ("x", "dt")] + [v["A"]] + [v[k][:, 0] for k in ("B", "C")]
    for idx in (torch.tensor([-1, 1, 3, 1 << 40], device=cuda_device),
                torch.tensor([-1, 1, 3, 7], dtype=torch.int32, device=cuda_device)):
        pool.copy_(before)
        y = selective_scan_step(*args, dt_softplus=True, state=pool, state_indices=idx)
        assert not y[[0, 2, 3]].any() and y[1].any()
        assert torch.equal(pool[[0, 2]], before[[0, 2]]) and not torch.equal(pool[1], before[1])
    assert pool._version > version
    assert not selective_scan_step(*args, state=pool[:0], state_indices=idx).any()


def test_steps_follow_the_scan(cuda_device):
    v = inputs(cuda_device, 3, 12, 24, 16, F32, F32, 3, seed=19)
    with torch.no_grad():
        y, ht = run(v)
    pool = v["h0"].clone()
    for t in range(12):
        yt = selective_scan_step(v["x"][:, t], v["dt"][:, t], v["A"], v["B"][:, t], v["C"][:, t], v["D"],
                                 v["z"][:, t], dt_bias=v["dt_bias"], dt_softplus=True, state=pool)
        close(yt, np64(y[:, t]))
    close(pool, np64(ht))


def test_captured_training_and_serving(cuda_device):
    """Forward, backward and a step in graphs, replayed on new inputs."""
    v = inputs(cuda_device, 2, 200, 24, 16, BF, F32, 2, seed=20)
    leaves = [v[k].requires_grad_() for k in NAMES]

    def step():
        y, ht = run(v)
        # no autograd graph of the leaves outlives its step
        return (y.detach(), ht.detach(), *torch.autograd.grad((y, ht), leaves, (v["dy"], v["dht"])))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            warm = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(warm, step()))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    w = inputs(cuda_device, 2, 200, 24, 16, BF, F32, 2, seed=21)
    with torch.no_grad():
        for k, t in v.items():
            t.copy_(w[k])
    g.replay()
    want = step()
    assert all(torch.equal(a, b) for a, b in zip(out, want))
    del g


def test_refusals(cuda_device):
    v = inputs(cuda_device, 2, 10, 12, 16, BF, BF, 2, seed=22)
    a = lambda **kw: [{**v, **kw}[k] for k in ("x", "dt", "A", "B", "C", "D", "z")]
    scan = lambda *p, **kw: selective_scan(*a(**kw), dt_bias=v["dt_bias"])
    for kw, err in ((dict(x=v["x"].cpu()), RuntimeError), (dict(dt=v["dt"][:, :5]), ValueError),
                    (dict(A=v["A"][:5]), ValueError), (dict(A=v["A"][:, 0]), ValueError),
                    (dict(A=torch.ones(12, 65, device=cuda_device)), NotImplementedError),
                    (dict(B=v["B"][:, :, :5]), ValueError), (dict(C=v["C"].float()), NotImplementedError),
                    (dict(B=v["B"][:, :, None].expand(2, 10, 5, 16), C=v["C"][:, :, None].expand(2, 10, 5, 16)),
                     ValueError),
                    (dict(D=v["D"][:3]), ValueError), (dict(z=v["z"].float()), NotImplementedError),
                    (dict(dt=v["dt"].half()), NotImplementedError), (dict(x=v["x"].double()), TypeError)):
        with pytest.raises(err):
            scan(**kw)
    with pytest.raises(ValueError):
        selective_scan(*a(), cu_seqlens=torch.tensor([0, 10], device=cuda_device))
    with pytest.raises(TypeError):
        selective_scan(*a(), initial_state=v["h0"].half())
    with pytest.raises(ValueError):
        selective_scan(*a(), initial_state=v["h0"][:1])
    pool = torch.zeros(2, 12, 16, device=cuda_device)
    one = lambda **kw: selective_scan_step(
        *[t[:, 0] if k not in ("A", "D") else t for k, t in zip(("x", "dt", "A", "B", "C", "D", "z"), a())], **kw)
    one(state=pool)
    for kw, err in ((dict(state=pool.half()), TypeError), (dict(state=pool[:1]), ValueError),
                    (dict(state=pool[:, :5]), ValueError), (dict(state=pool.transpose(1, 2)), ValueError),
                    (dict(state=pool, state_indices=torch.zeros(3, dtype=torch.int64)), ValueError),
                    (dict(state=pool.repeat(1, 1, 2)[:, :, :16]), ValueError)):
        with pytest.raises(err):
            one(**kw)


def test_forward_mode_is_refused(cuda_device):
    import torch.autograd.forward_ad as fwAD

    v = inputs(cuda_device, 1, 5, 4, 4, F32, F32, 1, seed=23)
    with fwAD.dual_level(), pytest.raises(Exception):
        run({**v, "x": fwAD.make_dual(v["x"], torch.ones_like(v["x"]))})
