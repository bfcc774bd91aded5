"""Arguments that the C entries of the selective scan, the token sampling and the
gradient norm refuse before any CUDA call (no GPU)."""

import ctypes
import math
import struct

import pytest

from qwendopamine_b200 import _native as N

F = ctypes.c_void_p(0x1000)


@pytest.fixture(scope="module")
def lib():
    return N.load()


def sel(**kw):
    base = dict(B=2, D=64, G=1, N=16, T=100, dtype=1, dt_dtype=0, dt_softplus=1, n_seqs=2, cu_seqlens=None,
                ld_x=64, ld_dt=64, ld_z=64, ld_b=16, ld_c=16, ld_dy=64)
    return N.SelectiveProblem(**{**base, **kw})


def fwd(lib, p, ws=None, size=0, saved=None, y=F):
    return lib.gdn2_selective_fwd(p, F, F, F, F, F, None, None, None, None, y, None, saved, ws, size, None)


def bwd(lib, p, ws=F, size=1 << 40):
    return lib.gdn2_selective_bwd(p, F, F, F, F, F, None, None, None, None, F, F, None, F, F, F, F, F, None, None,
                                  None, None, ws, size, None)


@pytest.mark.parametrize("kw,status", [
    (dict(D=0), N.ERR_INVALID), (dict(N=0), N.ERR_INVALID), (dict(G=0), N.ERR_INVALID),
    (dict(G=3), N.ERR_INVALID), (dict(N=65, ld_b=65, ld_c=65), N.ERR_UNSUPPORTED), (dict(dtype=5), N.ERR_INVALID),
    (dict(dt_dtype=2), N.ERR_UNSUPPORTED), (dict(n_seqs=3), N.ERR_INVALID), (dict(cu_seqlens=0x1000), N.ERR_INVALID),
    (dict(B=1, n_seqs=0, cu_seqlens=0x1000), N.ERR_INVALID), (dict(ld_x=63), N.ERR_INVALID),
    (dict(ld_dy=(1 << 22) + 1), N.ERR_INVALID), (dict(ld_c=15), N.ERR_INVALID), (dict(T=1 << 31), N.ERR_UNSUPPORTED),
    (dict(B=-1), N.ERR_INVALID), (dict(T=-1), N.ERR_INVALID)])
def test_selective_problems(lib, kw, status):
    p = sel(**kw)
    assert fwd(lib, p) == status and bwd(lib, p) == status
    assert lib.gdn2_selective_saved_bytes(p) == 0 and lib.gdn2_selective_workspace_bytes(p, 1) == 0
    one = sel(**{"T": 1, **kw})
    assert lib.gdn2_selective_step(one, F, F, F, F, F, None, None, None, F, 1024, 2, None, F, None) == status


def test_selective_pointers_and_workspaces(lib):
    p = sel()
    assert fwd(lib, p, y=None) == N.ERR_INVALID
    need = lib.gdn2_selective_workspace_bytes(p, 0)
    assert need > 0  # few channels: the time axis is cut
    assert fwd(lib, p) == N.ERR_WORKSPACE and fwd(lib, p, F, need - 1) == N.ERR_WORKSPACE
    assert fwd(lib, p, ctypes.c_void_p(0x1008), need) == N.ERR_INVALID
    assert fwd(lib, p, F, need, ctypes.c_void_p(0x1004)) == N.ERR_INVALID
    assert bwd(lib, p, None, 0) == N.ERR_WORKSPACE
    # 7 blocks of 16 rows for each entry, 16 states in fp32
    assert lib.gdn2_selective_saved_bytes(p) == 2 * 7 * 64 * 16 * 4
    assert lib.gdn2_selective_saved_bytes(sel(N=5, ld_b=5, ld_c=5)) == 2 * 7 * 64 * 8 * 4
    many = sel(B=1 << 20, n_seqs=1 << 20, D=1 << 20, T=1, ld_x=1 << 20, ld_dt=1 << 20, ld_z=1 << 20, ld_dy=1 << 20)
    assert fwd(lib, many) == N.ERR_UNSUPPORTED


def test_selective_step(lib):
    step = lambda p, state=F, stride=1024, pool=2, idx=None, y=F: lib.gdn2_selective_step(
        p, F, F, F, F, F, None, None, None, state, stride, pool, idx, y, None)
    p = sel(T=1)
    assert step(sel()) == N.ERR_INVALID  # more than one token
    assert step(p, state=None) == N.ERR_INVALID and step(p, y=None) == N.ERR_INVALID
    assert step(p, stride=1023) == N.ERR_INVALID and step(p, pool=1) == N.ERR_INVALID
    assert step(sel(T=1, B=0, n_seqs=0)) == N.OK


def test_selective_pointers_off_their_elements(lib):
    """Each pointer in turn one byte off: refused in front of any CUDA call."""
    odd = ctypes.c_void_p(0x1001)
    p = sel()
    for i in range(12):  # x dt A B C D z dt_bias h0 y ht saved
        args = [odd if k == i else F for k in range(12)]
        assert lib.gdn2_selective_fwd(p, *args, F, 1 << 40, None) == N.ERR_INVALID, i
    for i in range(21):  # the inputs to h0, saved, dy, dht, then the gradients
        args = [odd if k == i else F for k in range(21)]
        assert lib.gdn2_selective_bwd(p, *args, F, 1 << 40, None) == N.ERR_INVALID, i
    one = sel(T=1)
    for i in (0, 1, 2, 3, 4, 5, 6, 7, 8, 11, 12):
        args = [odd if k == i else F for k in range(13)]
        args[9], args[10] = 1024, 2
        assert lib.gdn2_selective_step(one, *args, None) == N.ERR_INVALID, i


def sample(**kw):
    base = dict(rows=4, ld=1000, vocab=1000, dtype=1, top_k=0, temperature=1.0, top_p=1.0, min_p=0.0)
    return N.SampleProblem(**{**base, **kw})


@pytest.mark.parametrize("kw", [dict(rows=-1), dict(vocab=0), dict(dtype=3), dict(ld=999), dict(top_k=-1),
                                dict(temperature=-1.0), dict(temperature=math.inf), dict(temperature=math.nan),
                                dict(top_p=-0.1), dict(top_p=1.1), dict(min_p=2.0), dict(min_p=math.nan)])
def test_sample_problems(lib, kw):
    assert lib.gdn2_sample(sample(**kw), F, F, None, None, None, None, F, None) == N.ERR_INVALID


def test_sample_pointers_and_sizes(lib):
    call = lambda p, x=F, u=F, ids=F: lib.gdn2_sample(p, x, u, None, None, None, None, ids, None)
    assert call(sample(rows=0), None, None, None) == N.OK
    for bad in (dict(x=None), dict(u=None), dict(ids=None), dict(x=ctypes.c_void_p(0x1001))):
        assert call(sample(), **bad) == N.ERR_INVALID
    assert call(sample(rows=1 << 30)) == N.ERR_UNSUPPORTED
    odd = ctypes.c_void_p(0x1002)
    for i in range(6):  # uniform temperature top_k top_p min_p token_ids
        args = [odd if k == i else F for k in range(6)]
        assert lib.gdn2_sample(sample(), F, *args, None) == N.ERR_INVALID, i


def table(*rows):
    return struct.pack(f"{3 * len(rows)}q", *(v for row in rows for v in row))


def test_gradient_norm(lib):
    norm = lambda t, n, kind=2, limit=1.0, out=F, ws=F, size=1 << 20: lib.gdn2_grad_norm(
        N.GradProblem(kind, limit), t, n, out, ws, size, None)
    good = table((0x1000, 10, 0))
    assert norm(good, -1) == N.ERR_INVALID and norm(None, 1) == N.ERR_INVALID
    assert norm(good, 1, kind=1) == N.ERR_INVALID and norm(good, 1, limit=math.nan) == N.ERR_INVALID
    assert norm(good, 1, out=None) == N.ERR_INVALID
    assert norm(good, 1, ws=None) == N.ERR_WORKSPACE and norm(good, 1, size=100) == N.ERR_WORKSPACE
    assert norm(good, 1, ws=ctypes.c_void_p(0x1004)) == N.ERR_INVALID
    assert norm(good, 1, out=ctypes.c_void_p(0x1002)) == N.ERR_INVALID
    assert lib.gdn2_grad_scale(good, 1, ctypes.c_void_p(0x1002), None) == N.ERR_INVALID
    for bad, status in ((( 0x1000, -1, 0), N.ERR_INVALID), ((0, 10, 0), N.ERR_INVALID), ((0x1000, 10, 3), N.ERR_INVALID),
                        ((0x1002, 10, 0), N.ERR_INVALID), ((0x1001, 10, 1), N.ERR_INVALID),
                        ((0x1000, 1 << 50, 0), N.ERR_UNSUPPORTED)):
        assert norm(table(bad), 1) == status
        assert lib.gdn2_grad_scale(table(bad), 1, F, None) == status
    assert lib.gdn2_grad_norm_workspace_bytes(-1) == 0
    assert lib.gdn2_grad_norm_workspace_bytes(100) >= 8 * 100


def test_scaled_tensors_that_share_memory(lib):
    scale = lambda *rows: lib.gdn2_grad_scale(table(*rows), len(rows), F, None)
    assert scale((0x1000, 10, 0), (0x1024, 10, 0)) == N.ERR_INVALID and b"overlap" in lib.gdn2_last_error()
    assert scale((0x2000, 8, 1), (0x1000, 3000, 1)) == N.ERR_INVALID
    assert scale((0x1000, 0, 0), (0, 0, 0)) == N.OK  # nothing to scale
    assert lib.gdn2_grad_scale(table((0x1000, 10, 0)), 1, None, None) == N.ERR_INVALID
