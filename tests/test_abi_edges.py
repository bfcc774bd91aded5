"""Arguments of the operators around the mixer that the C entries refuse before
any CUDA call (no GPU)."""

import ctypes

import pytest

from qwendopamine_b200 import _native as N


@pytest.fixture(scope="module")
def lib():
    return N.load()


def scan(**kw):
    base = dict(B=1, D=70, T=200, dtype=1, g_dtype=0, n_seqs=1, cu_seqlens=0x1000, ld_v=70,
                ld_g=70, ld_w=70, ld_dy=70)
    return N.ScanProblem(**{**base, **kw})


def test_scan_of_rows_without_a_sequence(lib):
    f = ctypes.c_void_p(0x1000)
    fwd = lambda p: lib.gdn2_scan_fwd(p, f, f, f, None, f, None, None, None)
    bwd = lambda p: lib.gdn2_scan_bwd(p, f, f, f, None, f, f, None, f, f, f, None, None)
    for call in (fwd, bwd):
        assert call(scan(n_seqs=0)) == N.ERR_INVALID and b"cu_seqlens" in lib.gdn2_last_error()
        assert call(scan(n_seqs=0, T=0)) == N.OK
    assert lib.gdn2_scan_saved_bytes(scan(n_seqs=0)) == 0


def test_logprob_temperature_without_an_inverse(lib):
    f = ctypes.c_void_p(0x1000)
    for t in (4e-39, 2.0 ** -149):
        p = N.LogprobProblem(4, 1000, -100, 1000, 1, 5, t)
        assert lib.gdn2_logprob_fwd(p, f, f, f, None, f, f, None, None) == N.ERR_INVALID
        assert b"temperature" in lib.gdn2_last_error()
        assert lib.gdn2_logprob_bwd(p, f, f, f, f, None, f, None) == N.ERR_INVALID
    none = N.LogprobProblem(0, 1000, -100, 1000, 1, 5, 1e-38)
    assert lib.gdn2_logprob_fwd(none, None, None, None, None, None, None, None, None) == N.OK
