"""Gated linear recurrence on B200: the diagonal sibling of the GDN-2 core.

Per channel, ``h_t = exp(g_t) h_{t-1} + w_t v_t`` and ``y_t = h_t`` -- GDN-2's
log-decay ``g`` and write gate ``w`` without keys, so a mixer built on it
shares the projections, the cache layout and the packing conventions.

* :func:`gated_scan` -- whole sequences: fixed length ``[B, T, ...]`` or packed
  ``[1, T, ...]`` with ``cu_seqlens``, fp32 states in and out, differentiable.
* :func:`gated_scan_step` -- one token per sequence on a pool of fp32 states
  that is updated in place (serving).

One launch of ``libgdn2_b200.so`` each (``gdn2_scan_fwd`` / ``gdn2_scan_bwd`` /
``gdn2_scan_step``); there is no CPU path.
"""

from __future__ import annotations

import math

import torch
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from .. import _native as N

__all__ = ["GatedScanFunction", "gated_scan", "gated_scan_step"]

MAX_STRIDE = 1 << 22  # of rows, in elements (the C entries refuse more)


def _rows(x, B, T, D):
    """``x`` as rows ``[B*T, D]`` with one row stride, and that stride; copied
    only when its strides are not those of such a matrix (a slice of a fused
    projection is)."""
    if x.is_contiguous():
        return x, D
    x = x.reshape(B, T, D)
    sb, st, sd = x.stride()
    if T == 1:
        st = sb
    elif B > 1 and sb != T * st:
        st = -1
    if (sd != 1 and D > 1) or (B * T > 1 and st < D) or st > MAX_STRIDE:
        return x.contiguous(), D
    return x, max(st, D)


class _Geometry:
    """Sizes, packing and row strides of one problem."""

    def __init__(self, v, g, w, cu):
        self.B, self.T = v.shape[0], v.shape[1]
        self.D = _width(v.shape[2:])
        self.n = self.B if cu is None else cu.numel() - 1
        self.v, self.ldv = _rows(v, self.B, self.T, self.D)
        self.g, self.ldg = _rows(g, self.B, self.T, self.D)
        self.w, self.ldw = _rows(w, self.B, self.T, self.D) if w is not None else (None, self.D)
        self.cu = cu

    def problem(self, ld_dy=None):
        return N.ScanProblem(self.B, self.D, self.T, N.dtype_code(self.v.dtype),
                             N.dtype_code(self.g.dtype), self.n, N.addr(self.cu), self.ldv,
                             self.ldg, self.ldw, self.D if ld_dy is None else ld_dy)


_width = math.prod  # elements of a shape


def _forward(geo, shape, h0, want_final, keep):
    lib = N.load()
    dev = geo.v.device
    prob = geo.problem()
    y = torch.empty(shape, dtype=geo.v.dtype, device=dev)
    ht = torch.empty(geo.n, geo.D, dtype=torch.float32, device=dev) if want_final else None
    saved = None
    if keep:
        saved = torch.empty(lib.gdn2_scan_saved_bytes(prob) // 4, dtype=torch.float32, device=dev)
    with N.on_device(dev.index):
        N.check(lib.gdn2_scan_fwd(prob, N.addr(geo.v), N.addr(geo.g), N.addr(geo.w), N.addr(h0),
                                  N.addr(y), N.addr(ht), N.addr(saved), N.raw_stream(dev.index)),
                "gdn2_scan_fwd")
    return y, ht, saved


class GatedScanFunction(torch.autograd.Function):
    """y, ht of :func:`gated_scan` with gradients for v, g, w and h0."""

    @staticmethod
    def forward(ctx, v, g, w, h0, cu, want_final):
        y, ht, saved = _forward(_Geometry(v, g, w, cu), v.shape, h0, want_final, keep=True)
        ctx.save_for_backward(v, g, w, h0, cu, saved)
        ctx.set_materialize_grads(False)
        return y, ht

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dht):
        v, g, w, h0, cu, saved = ctx.saved_tensors
        if dy is None and dht is None:
            return None, None, None, None, None, None
        lib = N.load()
        dev = v.device
        geo = _Geometry(v, g, w, cu)
        dy = torch.zeros_like(v) if dy is None else dy.to(v.dtype)
        dy, ld_dy = _rows(dy, geo.B, geo.T, geo.D)
        dht = dht.float().contiguous() if dht is not None else None
        prob = geo.problem(ld_dy)
        new = lambda x: torch.empty(x.shape, dtype=x.dtype, device=dev)
        dv, dg = new(v), new(g)
        dw = new(w) if w is not None else None
        dh0 = new(h0) if h0 is not None else None
        with N.on_device(dev.index):
            N.check(lib.gdn2_scan_bwd(prob, N.addr(geo.v), N.addr(geo.g), N.addr(geo.w), N.addr(h0),
                                      N.addr(saved), N.addr(dy), N.addr(dht), N.addr(dv),
                                      N.addr(dg), N.addr(dw), N.addr(dh0),
                                      N.raw_stream(dev.index)), "gdn2_scan_bwd")
        return dv, dg, dw, dh0, None, None


def _check(name, v, g, w, lead):
    for t in (v, g, w):
        if t is not None and not t.is_cuda:
            raise RuntimeError(f"{name}: inputs must be CUDA tensors -- the B200 build has no CPU "
                               "path")
    if v.ndim <= lead:
        raise ValueError(f"{name}: v needs at least {lead + 1} dimensions; got {tuple(v.shape)}")
    if _width(v.shape[lead:]) == 0:
        raise ValueError(f"{name}: v has no channels; got {tuple(v.shape)}")
    for n, t in (("g", g), ("w", w)):
        if t is not None and t.shape != v.shape:
            raise ValueError(f"{name}: {n} must have v's shape {tuple(v.shape)}; got "
                             f"{tuple(t.shape)}")
        if t is not None and t.device != v.device:
            raise ValueError(f"{name}: {n} is on {t.device}, v on {v.device}")
    N.dtype_code(v.dtype)
    if w is not None and w.dtype != v.dtype:
        raise NotImplementedError(f"{name}: v ({v.dtype}) and w ({w.dtype}) must share a dtype")
    if g.dtype != v.dtype and g.dtype != torch.float32:
        raise NotImplementedError(f"{name}: g ({g.dtype}) must be float32 or v's dtype ({v.dtype})")


def gated_scan(
    v: torch.Tensor,
    g: torch.Tensor,
    w: torch.Tensor | None = None,
    initial_state: torch.Tensor | None = None,
    output_final_state: bool = False,
    cu_seqlens: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    r"""``h_t = exp(g_t) h_{t-1} + w_t v_t`` over the second dimension.

    v: ``[B, T, ...]`` (float32, bfloat16 or float16); g, the log-decay, of
    v's shape in float32 or v's dtype (-inf cuts the past off; positive values
    grow the state, as long as the product of the decays of 128 rows stays
    finite in float32, also where the state is zero); w of v's shape and dtype, or None for ones.
    ``initial_state`` and the returned final state (None unless
    ``output_final_state``) are float32 ``[N, ...]``.  With ``cu_seqlens``
    (``[N+1]``, from 0 to T, not decreasing; not checked on the device) B must
    be 1 and the N packed sequences, empty ones included, each start from
    their own state; N = B otherwise.  Returns ``(y, final_state)``, y in v's
    dtype; states and sums are float32.  Differentiable (once) in v, g, w and
    ``initial_state``, in reverse mode; the gradients need no forward value but
    a state every 64 tokens.  Rows may be strided (slices of a fused projection).
    """
    _check("gated_scan", v, g, w, 2)
    n = v.shape[0]
    cu = None
    if cu_seqlens is not None:
        if v.shape[0] != 1:
            raise ValueError(
                f"The batch size is expected to be 1 rather than {v.shape[0]} when using "
                "`cu_seqlens`. Please flatten variable-length inputs before processing.")
        if cu_seqlens.ndim != 1 or cu_seqlens.numel() < 1 or cu_seqlens.is_floating_point():
            raise ValueError("cu_seqlens must be a 1-D tensor of offsets")
        n = cu_seqlens.numel() - 1
    if n > N.INT32_MAX:
        raise ValueError(f"gated_scan: up to 2^31 - 1 sequences are supported; got {n}")
    if cu_seqlens is not None:
        cu = cu_seqlens.to(device=v.device, dtype=torch.int32).contiguous()
    h0 = initial_state
    if h0 is not None:
        if h0.dtype != torch.float32:
            raise TypeError("initial_state must be in float32.")
        if h0.device != v.device or tuple(h0.shape) != (n, *v.shape[2:]):
            raise ValueError(f"initial_state must be [{n}, *{tuple(v.shape[2:])}] on {v.device}; "
                             f"got {tuple(h0.shape)} on {h0.device}")
        h0 = h0.contiguous()
    if N.forward_mode(v, g, w, h0) or torch.is_grad_enabled() and any(
            t is not None and t.requires_grad for t in (v, g, w, h0)):
        y, ht = GatedScanFunction.apply(v, g, w, h0, cu, bool(output_final_state))
    else:
        y, ht, _ = _forward(_Geometry(v, g, w, cu), v.shape, h0, bool(output_final_state),
                            keep=False)
    return y, ht.view(n, *v.shape[2:]) if ht is not None and v.ndim > 3 else ht


def gated_scan_step(
    v: torch.Tensor,
    g: torch.Tensor,
    w: torch.Tensor | None = None,
    *,
    state: torch.Tensor,
    state_indices: torch.Tensor | None = None,
) -> torch.Tensor:
    r"""One token for each of N sequences (inference only).

    v, g, w: ``[N, ...]`` as in :func:`gated_scan` without the time dimension.
    ``state``: float32 pool ``[S, ...]``, updated in place; sequence n uses
    row ``state_indices[n]`` (row n without indices).  An index outside
    ``[0, S)`` marks padding: no state changes and its row of y is zero.  Two
    sequences must not name the same row.  Returns y ``[N, ...]`` in v's dtype.
    """
    _check("gated_scan_step", v, g, w, 1)
    n, D = v.shape[0], _width(v.shape[1:])
    if state.dtype != torch.float32:
        raise TypeError("state must be in float32.")
    if state.device != v.device or state.shape[1:] != v.shape[1:]:
        raise ValueError(f"state must be [S, *{tuple(v.shape[1:])}] on {v.device}; got "
                         f"{tuple(state.shape)} on {state.device}")
    if n > N.INT32_MAX or state.shape[0] > N.INT32_MAX:
        raise ValueError(f"gated_scan_step: up to 2^31 - 1 sequences and states are supported; got "
                         f"{n} and {state.shape[0]}")
    if not state.is_contiguous() and (not state[:1].is_contiguous() or (
            state.shape[0] > 1 and state.stride(0) < D)):
        raise ValueError("state must hold each sequence's channels contiguously")
    idx = None
    if state_indices is not None:
        if state_indices.shape != (n,) or state_indices.is_floating_point():
            raise ValueError(f"state_indices must be {n} integers; got "
                             f"{tuple(state_indices.shape)} {state_indices.dtype}")
        idx = state_indices
        if idx.dtype is not torch.int32:  # outside the pool stays outside in 32 bits
            idx = idx.to(torch.int64).clamp(-1, state.shape[0]).to(torch.int32)
        idx = idx.to(v.device).contiguous()
    elif state.shape[0] < n:
        raise ValueError(f"{n} sequences need as many states; got {state.shape[0]}")
    y = torch.empty(v.shape, dtype=v.dtype, device=v.device)
    if n == 0:
        return y
    if state.shape[0] == 0:
        return y.zero_()
    (v, ldv), (g, ldg) = _rows(v, n, 1, D), _rows(g, n, 1, D)
    w, ldw = _rows(w, n, 1, D) if w is not None else (None, D)
    prob = N.ScanProblem(n, D, 1, N.dtype_code(v.dtype), N.dtype_code(g.dtype), n, None, ldv, ldg,
                         ldw, D)
    index = v.device.index
    with N.on_device(index):
        N.check(N.load().gdn2_scan_step(
            prob, N.addr(v), N.addr(g), N.addr(w), N.addr(state), max(state.stride(0), D),
            state.shape[0], N.addr(idx), N.addr(y), N.raw_stream(index)), "gdn2_scan_step")
    increment_version(state)  # autograd does not see the kernel's writes
    return y
