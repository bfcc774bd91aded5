"""Gated linear recurrence on the GPU: calls at the edges of what the entry
points take."""

import threading

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from qwendopamine_b200 import _native as N
from qwendopamine_b200 import gated_scan, gated_scan_step

pytestmark = pytest.mark.gpu

F32, BF = torch.float32, torch.bfloat16


def inputs(dev, B, T, D, dtype, gdtype, gate, n, seed=0):
    gen = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen)
    return dict(v=rn(B, T, D).to(dev, dtype),
                g=torch.nn.functional.logsigmoid(rn(B, T, D) + 3).to(dev, gdtype),
                w=torch.sigmoid(rn(B, T, D)).to(dev, dtype) if gate else None,
                h0=rn(n, D).to(dev))


def test_shapes_of_several_host_threads(cuda_device):
    """One kernel serves a long sequence (a cluster of CTAs, more shared memory)
    and short ones (single CTAs) from several host threads at once."""
    lib, D = N.load(), 40
    calls, errors, start = [], [], threading.Barrier(4)
    for i, T in enumerate((2000, 300, 2000, 300)):
        x = inputs(cuda_device, 1, T, D, F32, F32, True, 1, seed=20 + i)
        want, _ = gated_scan(x["v"], x["g"], x["w"])
        calls.append((x, want, torch.empty_like(want), torch.cuda.Stream()))
    torch.cuda.synchronize()

    def work(x, want, y, stream):
        T = want.shape[1]
        prob = N.ScanProblem(1, D, T, N.dtype_code(F32), N.dtype_code(F32), 1, None, D, D, D, D)
        args = (prob, *(x[k].data_ptr() for k in ("v", "g", "w")), None, y.data_ptr(), None, None,
                stream.cuda_stream)
        start.wait()
        try:
            for _ in range(20000):
                N.check(lib.gdn2_scan_fwd(*args), "gdn2_scan_fwd")
            stream.synchronize()
            assert torch.equal(y, want)
        except Exception as e:
            errors.append(e)

    threads = [threading.Thread(target=work, args=a) for a in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


def test_step_marks_the_pool_as_changed(cuda_device):
    """A graph that saved the states cannot be differentiated after a step on them."""
    x = inputs(cuda_device, 3, 1, 16, F32, F32, False, 3, seed=22)
    pool = x["h0"].clone()
    leaf = torch.ones(3, 16, device=cuda_device, requires_grad=True)
    loss = (leaf * pool).sum()
    version = pool._version
    gated_scan_step(x["v"][:, 0], x["g"][:, 0], state=pool)
    assert pool._version > version
    with pytest.raises(RuntimeError, match="inplace operation"):
        loss.backward()
    with torch.inference_mode():  # tensors without a version
        own = torch.zeros(3, 16, device=cuda_device)
        y = gated_scan_step(x["v"][:, 0], x["g"][:, 0], state=own)
        assert torch.equal(y, own)


@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused(cuda_device, grad):
    """No tangent is lost without a word, also where nothing requires a gradient."""
    x = inputs(cuda_device, 1, 6, 8, F32, F32, True, 1, seed=23)
    names = ("v", "g", "w", "h0")
    plain, _ = gated_scan(x["v"], x["g"], x["w"], x["h0"])
    for name in names:
        with fwAD.dual_level(), torch.set_grad_enabled(grad):
            d = dict(x)
            d[name] = fwAD.make_dual(x[name], torch.ones_like(x[name]))
            with pytest.raises(RuntimeError, match="forward"):
                gated_scan(*(d[k] for k in names))
            y, _ = gated_scan(*(x[k] for k in names))  # no tangents: as ever
            assert torch.equal(y, plain)


@pytest.mark.parametrize("itype", [torch.int64, torch.int32])
def test_wide_indices_outside_the_pool_are_padding(cuda_device, itype):
    """Sentinels that do not fit 32 bits mark padding like any other index
    outside the pool."""
    far = [torch.iinfo(itype).min, torch.iinfo(itype).max, -1, 4]
    if itype == torch.int64:
        far += [1 << 32, (1 << 32) + 1, -(1 << 32), (1 << 31) + 1]
    n, D = len(far) + 1, 40
    x = inputs(cuda_device, n, 1, D, F32, F32, False, n, seed=21)
    v, g = x["v"][:, 0], x["g"][:, 0]
    pool = torch.randn(4, D, device=cuda_device)
    before = pool.clone()
    idx = torch.tensor(far + [3], dtype=itype, device=cuda_device)
    y = gated_scan_step(v, g, state=pool, state_indices=idx)
    assert torch.equal(pool[:3], before[:3]) and not torch.equal(pool[3], before[3])
    assert not y[:-1].any() and torch.equal(y[-1], pool[3])
    # indices on the host give the same
    y2 = gated_scan_step(v[-1:], g[-1:], state=before, state_indices=idx[-1:].cpu())
    assert torch.equal(y2, y[-1:]) and torch.equal(before, pool)


def test_rows_without_a_sequence_are_refused(cuda_device):
    """Offsets without a sequence cannot end at the last of some rows."""
    v = torch.ones(1, 5, 8, device=cuda_device)
    cu = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    with pytest.raises(ValueError, match="cu_seqlens"):
        gated_scan(v, -v, cu_seqlens=cu)
    y, ht = gated_scan(v[:, :0], v[:, :0], cu_seqlens=cu, output_final_state=True)
    assert y.shape == (1, 0, 8) and ht.shape == (0, 8)


def fault_word():
    return N.load().gdn2_fault_status(None, 1)


@pytest.mark.parametrize("dtype,gdtype", [(F32, F32), (BF, F32)])
@pytest.mark.parametrize("T,D", [(40000, 64), (700, 20), (9001, 1000)])
def test_bounded_wait_runs_out_cleanly(cuda_device, T, D, dtype, gdtype):
    """The failure path of the exchange between a cluster's CTAs, made to happen
    without a fault: every CTA waits for more than comes, 50 us at most.  The
    launch succeeds, bit 4 of the fault word is set, all results are NaN, and the
    next call on the same context is as good as ever."""
    lib = N.load()
    fault_word()
    x = inputs(cuda_device, 1, T, D, dtype, gdtype, False, 1, seed=30)
    v, g = x["v"], x["g"]
    prob = N.ScanProblem(1, D, T, N.dtype_code(dtype), N.dtype_code(gdtype), 1, None, D, D, D, D)
    saved, lost = (torch.zeros(lib.gdn2_scan_saved_bytes(prob) // 4, device=cuda_device)
                   for _ in range(2))
    y, y2, dy, dv, dv2 = (torch.zeros_like(v) for _ in range(5))
    dg, dg2 = torch.zeros_like(g), torch.zeros_like(g)
    dy.copy_(torch.randn(v.shape, generator=torch.Generator().manual_seed(31)))
    a, st = (lambda t: t.data_ptr()), N.raw_stream(0)

    def normal():
        N.check(lib.gdn2_scan_fwd(prob, a(v), a(g), None, None, a(y), None, a(saved), st), "fwd")
        N.check(lib.gdn2_scan_bwd(prob, a(v), a(g), None, None, a(saved), a(dy), None, a(dv), a(dg),
                                  None, None, st), "bwd")

    normal()
    want = [t.clone() for t in (y, saved, dv, dg)]
    N.check(lib.gdn2_test_scan_wait_timeout(prob, a(v), a(g), a(y2), a(lost), None, None, None,
                                            50_000, st), "fwd")
    assert fault_word() == 16
    used = -(-T // 64) * D  # a state for every 64 rows
    assert y2.isnan().all() and lost[:used].isnan().all() and not lost[used:].any()
    N.check(lib.gdn2_test_scan_wait_timeout(prob, a(v), a(g), None, a(saved), a(dy), a(dv2), a(dg2),
                                            50_000, st), "bwd")
    assert fault_word() == 16
    assert dv2.isnan().all() and dg2.isnan().all()
    for t in (y, dv, dg):
        t.zero_()
    normal()
    assert fault_word() == 0
    assert all(torch.equal(t, w) for t, w in zip((y, saved, dv, dg), want))


def test_wait_hook_argument_checks(cuda_device):
    lib, buf = N.load(), torch.zeros(4, 20, device=cuda_device)
    one = N.ScanProblem(1, 20, 4, 0, 0, 1, None, 20, 20, 20, 20)
    a = buf.data_ptr()
    call = lambda p, ns: lib.gdn2_test_scan_wait_timeout(p, a, a, a, None, None, None, None, ns, None)
    for ns in (0, 2_000_000_000):
        assert call(one, ns) == N.ERR_INVALID
    assert call(one, 1000) == N.ERR_CUDA and b"not supported" in lib.gdn2_last_error()
    assert lib.gdn2_fault_status(None, 1) == 0


def test_sizes_beyond_32_bits_are_refused(cuda_device):
    """The library holds these sizes in 32 bits; the rows are one row, expanded."""
    many = (1 << 32) + 1
    one = torch.zeros(1, 1, 1, device=cuda_device)
    with pytest.raises(ValueError, match="2.31 - 1 sequences"):
        gated_scan(one.expand(many, 1, 1), one.expand(many, 1, 1))
    with pytest.raises(ValueError, match="2.31 - 1 sequences"):
        gated_scan(one, one, cu_seqlens=torch.zeros(1, device=cuda_device).int().expand(many + 1))
    with pytest.raises(ValueError, match="2.31 - 1 sequences"):
        gated_scan_step(one[0].expand(many, 1), one[0].expand(many, 1), state=one[0])
    with pytest.raises(ValueError, match="2.31 - 1 sequences and states"):
        gated_scan_step(one[0], one[0], state=one[0].expand(many, 1))


def test_capture_in_a_graph(cuda_device):
    """Forward, backward and step replayed on new inputs in the captured buffers."""
    x = inputs(cuda_device, 2, 300, 40, BF, F32, True, 2, seed=24)
    leaves = [x[k].requires_grad_() for k in ("v", "g", "w", "h0")]
    dy, dht = torch.randn_like(x["v"]), torch.randn_like(x["h0"])
    pool = torch.randn(2, 40, device=cuda_device)
    slots = torch.tensor([1, 0], device=cuda_device)

    def go():
        y, ht = gated_scan(*leaves[:3], initial_state=leaves[3], output_final_state=True)
        grads = torch.autograd.grad((y, ht), leaves, (dy, dht))
        with torch.no_grad():
            one = gated_scan_step(*(t[:, 0] for t in leaves[:3]), state=pool, state_indices=slots)
        return (y, ht, *grads, one)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        go()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = go()
    other = inputs(cuda_device, 2, 300, 40, BF, F32, True, 2, seed=25)
    with torch.no_grad():
        for leaf, k in zip(leaves, ("v", "g", "w", "h0")):
            leaf.copy_(other[k])
    before = pool.clone()
    graph.replay()
    got, moved = [t.clone() for t in out], pool.clone()
    pool.copy_(before)
    for a, b in zip(got, go()):
        assert torch.equal(a, b)
    assert torch.equal(moved, pool)
