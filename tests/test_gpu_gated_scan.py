"""Gated linear recurrence on the GPU against the float64 oracle.

Tolerances (relative L2).  fp32 results: each step rounds the decay (2 ulp of
expf), a product and a sum, about 3 * 2^-24 per step, over the effective
window of at most a few hundred steps that these decays leave: 2e-5.  16-bit
results: one rounding of a value that is right to fp32, at most 2^-9 (bf16) or
2^-12 (fp16) of each element; twice that.  States and the gradients of fp32
inputs are fp32 results whatever the token type.
"""

import numpy as np
import pytest
import torch

from oracle import op_oracle as O
from qwendopamine_b200 import gated_scan, gated_scan_step

pytestmark = pytest.mark.gpu

TOL = {torch.float32: 2e-5, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
F32, BF, FH = torch.float32, torch.bfloat16, torch.float16


def np64(t):
    return None if t is None else t.detach().double().cpu().numpy()


def close(got, want, dtype=None):
    a = np64(got)
    assert a.shape == want.shape
    assert np.isfinite(a).all()
    err = np.linalg.norm(a - want) / max(np.linalg.norm(want), 1e-30)
    assert err <= TOL[dtype or got.dtype], err


def inputs(dev, B, T, D, dtype, gdtype, gate, n, seed=0, decay=None):
    gen = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen)
    g = torch.nn.functional.logsigmoid(rn(B, T, D) + 3) if decay is None else decay(rn(B, T, D))
    v, dy = rn(B, T, D).to(dev, dtype), rn(B, T, D).to(dev, dtype)
    w = torch.sigmoid(rn(B, T, D)).to(dev, dtype) if gate else None
    return dict(v=v, g=g.to(dev, gdtype), w=w, h0=rn(n, D).to(dev), dy=dy, dht=rn(n, D).to(dev))


def check(x, cu=None, use_h0=True, use_dht=True):
    leaves = {k: x[k].detach().requires_grad_() for k in ("v", "g", "w", "h0")
              if x[k] is not None and (k != "h0" or use_h0)}
    cut = None if cu is None else torch.tensor(cu, dtype=torch.int32, device=x["v"].device)
    y, ht = gated_scan(leaves["v"], leaves["g"], leaves.get("w"),
                       initial_state=leaves.get("h0"), output_final_state=True, cu_seqlens=cut)
    outs, gout = [y], [x["dy"]]
    if use_dht:
        outs.append(ht)
        gout.append(x["dht"])
    grads = dict(zip(leaves, torch.autograd.grad(outs, list(leaves.values()), gout)))
    with torch.no_grad():
        y2, ht2 = gated_scan(x["v"], x["g"], x["w"], initial_state=x["h0"] if use_h0 else None,
                             output_final_state=True, cu_seqlens=cut)
    assert torch.equal(y, y2) and torch.equal(ht, ht2)
    a = [np64(x[k]) for k in ("v", "g", "w")] + [np64(x["h0"]) if use_h0 else None]
    ry, rh = O.scan_fwd(*a, cu)
    close(y, ry)
    close(ht, rh)
    want = dict(zip(("v", "g", "w", "h0"),
                    O.scan_bwd(*a, np64(x["dy"]), np64(x["dht"]) if use_dht else None, cu)))
    for k, d in grads.items():
        assert d.dtype == x[k].dtype and d.shape == x[k].shape
        close(d, want[k])


TYPES = [(F32, F32, True), (BF, F32, True), (BF, BF, False), (FH, FH, True), (FH, F32, False)]


@pytest.mark.parametrize("dtype,gdtype,gate", TYPES)
@pytest.mark.parametrize("B,T,D", [(1, 1, 1), (5, 1, 64), (3, 5, 7), (1, 63, 64), (2, 64, 65),
                                   (2, 65, 128), (1, 129, 62), (2, 300, 200)])
def test_fixed_length(cuda_device, B, T, D, dtype, gdtype, gate):
    check(inputs(cuda_device, B, T, D, dtype, gdtype, gate, B))


@pytest.mark.parametrize("B,T,D", [(1, 9001, 20), (2, 4097, 66), (1, 8192, 64), (130, 100, 36)])
def test_long_scans_cross_groups_of_tiles(cuda_device, B, T, D):
    check(inputs(cuda_device, B, T, D, BF, F32, True, B, seed=1))


@pytest.mark.parametrize("dtype,gdtype,gate", TYPES)
def test_packed_sequences(cuda_device, dtype, gdtype, gate):
    lens = [0, 1, 5, 0, 0, 127, 128, 129, 1, 1000, 64, 0, 3000, 2, 0]
    cu = np.concatenate([[0], np.cumsum(lens)]).tolist()
    check(inputs(cuda_device, 1, cu[-1], 72, dtype, gdtype, gate, len(lens), seed=2), cu)


def test_no_start_state_and_no_end_gradient(cuda_device):
    x = inputs(cuda_device, 3, 200, 40, BF, F32, True, 3, seed=3)
    check(x, use_h0=False)
    check(x, use_dht=False)
    check(x, use_h0=False, use_dht=False)


def test_gradient_of_the_end_state_alone(cuda_device):
    x = inputs(cuda_device, 2, 150, 24, F32, F32, True, 2, seed=4)
    leaves = [x[k].requires_grad_() for k in ("v", "g", "w", "h0")]
    _, ht = gated_scan(*leaves[:3], initial_state=leaves[3], output_final_state=True)
    got = torch.autograd.grad(ht, leaves, x["dht"])
    want = O.scan_bwd(*(np64(t) for t in leaves), np.zeros((2, 150, 24)), np64(x["dht"]))
    for a, b in zip(got, want):
        close(a, b)


@pytest.mark.parametrize("decay", ["strong", "none", "reset", "growth", "slow"])
def test_extreme_decays(cuda_device, decay):
    f = {"strong": lambda z: -40 - z.abs(), "none": lambda z: z * 0,
         "reset": lambda z: torch.where(z > 1, -torch.inf, -0.1 * z.abs()),
         "growth": lambda z: 0.01 * z.abs(), "slow": lambda z: -0.01 * z.abs()}[decay]
    check(inputs(cuda_device, 2, 260, 48, F32, F32, True, 2, seed=5, decay=f))


def test_empty_batches_and_empty_sequences(cuda_device):
    h0 = torch.randn(3, 8, device=cuda_device)
    z = lambda *s: torch.zeros(*s, device=cuda_device)
    y, ht = gated_scan(z(3, 0, 8), z(3, 0, 8), initial_state=h0, output_final_state=True)
    assert y.shape == (3, 0, 8) and torch.equal(ht, h0)
    y, ht = gated_scan(z(0, 4, 8), z(0, 4, 8), output_final_state=True)
    assert y.shape == (0, 4, 8) and ht.shape == (0, 8)
    cu = torch.zeros(4, dtype=torch.int64, device=cuda_device)
    y, ht = gated_scan(z(1, 0, 8), z(1, 0, 8), initial_state=h0, output_final_state=True,
                       cu_seqlens=cu)
    assert torch.equal(ht, h0)
    leaf = h0.clone().requires_grad_()
    y, ht = gated_scan(z(1, 0, 8), z(1, 0, 8), initial_state=leaf, output_final_state=True,
                       cu_seqlens=cu)
    d, = torch.autograd.grad(ht, leaf, h0)
    assert torch.equal(d, h0)


def test_a_sequence_does_not_reach_the_next(cuda_device):
    lens = [70, 300, 65, 4200, 10]
    cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device=cuda_device)
    T = int(cu[-1])
    x = inputs(cuda_device, 1, T, 66, F32, F32, True, len(lens), seed=6)
    bad = {k: t.clone() if t is not None else None for k, t in x.items()}
    for n, val in ((0, float("nan")), (1, float("inf")), (3, float("nan"))):
        lo, hi = int(cu[n]), int(cu[n + 1])
        bad["v"][:, lo + 2:hi:7] = val
        bad["dy"][:, lo + 3:hi:5] = val
        bad["h0"][n] = val
        bad["dht"][n] = val

    def go(x):
        leaves = [x[k].detach().requires_grad_() for k in ("v", "g", "w", "h0")]
        y, ht = gated_scan(*leaves[:3], initial_state=leaves[3], output_final_state=True,
                           cu_seqlens=cu)
        return (y, ht, *torch.autograd.grad((y, ht), leaves, (x["dy"], x["dht"])))

    for a, b in zip(go(x), go(bad)):
        for n in (2, 4):
            lo, hi = int(cu[n]), int(cu[n + 1])
            if a.shape[0] == len(lens):
                assert torch.equal(a[n], b[n])
            else:
                assert torch.equal(a[0, lo:hi], b[0, lo:hi])


def test_strided_rows_and_views(cuda_device):
    """Slices of one fused projection, odd offsets, transposed and expanded inputs."""
    gen = torch.Generator().manual_seed(7)
    fused = torch.randn(2, 140, 3 * 48 + 3, generator=gen).to(cuda_device)
    for off in (0, 3):
        v, g, w = (fused[..., off + i * 48: off + (i + 1) * 48] for i in range(3))
        g = -g.abs()
        y, ht = gated_scan(v, g, w, output_final_state=True)
        yc, hc = gated_scan(v.contiguous(), g.contiguous(), w.contiguous(), output_final_state=True)
        assert torch.equal(y, yc) and torch.equal(ht, hc)
    t = torch.randn(140, 2, 48, generator=gen).to(cuda_device).transpose(0, 1)
    e = torch.full((2, 1, 1), -0.1, device=cuda_device).expand(2, 140, 48)
    y, _ = gated_scan(t, e)
    yc, _ = gated_scan(t.contiguous(), e.contiguous())
    assert torch.equal(y, yc)
    heads = torch.randn(2, 9, 3, 5, generator=gen).to(cuda_device)
    y, ht = gated_scan(heads, -heads.abs(), output_final_state=True)
    assert y.shape == heads.shape and ht.shape == (2, 3, 5)


def test_rows_far_apart(cuda_device):
    """A row stride beyond what a tile's 32-bit offsets hold."""
    far = torch.zeros(3, (1 << 22) + 8, device=cuda_device)
    x = inputs(cuda_device, 1, 3, 40, F32, F32, False, 1, seed=13)
    far[:, 3:43] = x["v"][0]
    y, _ = gated_scan(far[None, :, 3:43], x["g"])
    assert torch.equal(y, gated_scan(x["v"], x["g"])[0])


def test_offsets_beyond_32_bits(cuda_device):
    """More than 2^31 values: the last sequence is as good as the first."""
    B, T, D = 70, 16384, 1900
    v = torch.zeros(B, T, D, dtype=BF, device=cuda_device)
    g = torch.full((1, 1, 1), -0.01, dtype=BF, device=cuda_device).expand(B, T, D).contiguous()
    v[-1] = torch.randn(T, D, device=cuda_device).to(BF)
    v.requires_grad_()
    y, ht = gated_scan(v, g, output_final_state=True)
    ry, rh = O.scan_fwd(np64(v[-1:, :, :40]), np64(g[-1:, :, :40]))
    close(y[-1:, :, :40], ry)
    close(ht[-1:, :40], rh)
    assert not y[-2].any()
    dy = torch.zeros_like(v)
    dy[-1] = v[-1].detach()
    d, = torch.autograd.grad(y, v, dy)
    want = O.scan_bwd(np64(v[-1:, :, :40]), np64(g[-1:, :, :40]), None, None, np64(dy[-1:, :, :40]))
    close(d[-1:, :, :40], want[0])
    assert not d[-2].any()


def test_gradient_of_a_broadcast_decay(cuda_device):
    """One decay for a head's channels: the gradient sums over them."""
    x = inputs(cuda_device, 2, 90, 32, F32, F32, False, 2, seed=8)
    g1 = x["g"][..., :1].clone().requires_grad_()
    y, _ = gated_scan(x["v"], g1.expand(2, 90, 32))
    d, = torch.autograd.grad(y, g1, x["dy"])
    wide = np.broadcast_to(np64(g1), (2, 90, 32))
    dg = O.scan_bwd(np64(x["v"]), wide, None, None, np64(x["dy"]))[1]
    close(d, dg.sum(-1, keepdims=True))


def test_equal_inputs_give_equal_bits(cuda_device):
    x = inputs(cuda_device, 1, 20000, 256, BF, F32, True, 1, seed=9)

    def go():
        leaves = [x[k].detach().requires_grad_() for k in ("v", "g", "w", "h0")]
        y, ht = gated_scan(*leaves[:3], initial_state=leaves[3], output_final_state=True)
        return (y, ht, *torch.autograd.grad((y, ht), leaves, (x["dy"], x["dht"])))

    first = go()
    for _ in range(5):
        for a, b in zip(first, go()):
            assert torch.equal(a, b)


def test_another_stream(cuda_device):
    x = inputs(cuda_device, 2, 500, 64, BF, F32, True, 2, seed=10)
    want = gated_scan(x["v"], x["g"], x["w"], output_final_state=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = gated_scan(x["v"], x["g"], x["w"], output_final_state=True)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("dtype,gdtype,gate", TYPES)
@pytest.mark.parametrize("n,D", [(1, 1), (7, 66), (33, 256)])
def test_step_on_a_pool(cuda_device, n, D, dtype, gdtype, gate):
    x = inputs(cuda_device, n, 1, D, dtype, gdtype, gate, n, seed=11)
    tok = [x[k][:, 0] if x[k] is not None else None for k in ("v", "g", "w")]
    pool = torch.randn(n + 5, D, device=cuda_device)
    slots = torch.randperm(n + 5, device=cuda_device)[:n].to(torch.int32)
    if n > 2:
        slots[1], slots[2] = -1, n + 5  # padding
    used = [i for i in range(n) if 0 <= int(slots[i]) < n + 5]
    before = pool.clone()
    y = gated_scan_step(*tok, state=pool, state_indices=slots)
    want = before.clone().double().cpu().numpy()
    ry = np.zeros((n, D))
    for i in used:
        s = int(slots[i])
        h = np.exp(np64(tok[1])[i]) * want[s] + np64(tok[0])[i] * (1 if not gate else np64(tok[2])[i])
        want[s] = ry[i] = h
    close(y, ry)
    close(pool, want)
    left = [s for s in range(n + 5) if s not in {int(slots[i]) for i in used}]
    assert torch.equal(pool[left], before[left])


def test_step_continues_a_scan(cuda_device):
    x = inputs(cuda_device, 3, 20, 40, F32, F32, True, 3, seed=12)
    y, ht = gated_scan(x["v"], x["g"], x["w"], initial_state=x["h0"], output_final_state=True)
    pool = x["h0"].clone()
    for t in range(20):
        yt = gated_scan_step(x["v"][:, t], x["g"][:, t], x["w"][:, t], state=pool)
        close(yt, np64(y[:, t]))
    close(pool, np64(ht))
    wide = torch.zeros(3, 2, 40, device=cuda_device)  # a slice of a larger pool
    wide[:, 1] = x["h0"]
    yt = gated_scan_step(x["v"][:, 0], x["g"][:, 0], x["w"][:, 0], state=wide[:, 1])
    close(yt, np64(y[:, 0]))
    assert not wide[:, 0].any()


def test_refusals(cuda_device):
    z = lambda *s, **k: torch.zeros(*s, device=cuda_device, **k)
    v = z(2, 4, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        gated_scan(torch.zeros(1, 2, 8), torch.zeros(1, 2, 8))
    with pytest.raises(ValueError, match="g must have"):
        gated_scan(v, z(2, 4, 1))
    with pytest.raises(NotImplementedError, match="share a dtype"):
        gated_scan(v, v, z(2, 4, 8, dtype=BF))
    with pytest.raises(NotImplementedError, match="float32"):
        gated_scan(v, z(2, 4, 8, dtype=BF))
    with pytest.raises(TypeError):
        gated_scan(v.double(), v)
    with pytest.raises(ValueError, match="batch size"):
        gated_scan(v, v, cu_seqlens=torch.tensor([0, 4], device=cuda_device))
    with pytest.raises(ValueError, match="initial_state"):
        gated_scan(v, v, initial_state=z(3, 8))
    with pytest.raises(TypeError, match="float32"):
        gated_scan(v, v, initial_state=z(2, 8, dtype=BF))
    with pytest.raises(ValueError, match="no channels"):
        gated_scan(z(2, 4, 0), z(2, 4, 0))
    with pytest.raises(ValueError, match="as many states"):
        gated_scan_step(v[:, 0], v[:, 0], state=z(1, 8))
    with pytest.raises(ValueError, match="state must"):
        gated_scan_step(v[:, 0], v[:, 0], state=z(2, 9))
    with pytest.raises(ValueError, match="integers"):
        gated_scan_step(v[:, 0], v[:, 0], state=z(2, 8), state_indices=z(3, dtype=torch.int32))
    x = z(1, 3, 4).requires_grad_()
    y, _ = gated_scan(x, z(1, 3, 4))
    d, = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(d.sum(), x)
