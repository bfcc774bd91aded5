"""Selective state space scan on B200: the sibling of ``gated_scan`` with N states
for each channel.

Per channel d and state n, ``h_t = exp(dt_t A) h_{t-1} + dt_t x_t B_t`` and ``y_t =
(sum_n h_t C_t + D x_t) silu(z_t)``: decays and inputs depend on the token, and
the vectors B and C are shared by a group of channels.  In front of it stands the
block's short causal convolution (``short_conv``, for prompts and, with its prefix
and state, for single tokens; it knows no ``cu_seqlens``: packed sequences are
convolved one by one, or as the rows of a padded batch).

* :func:`selective_scan` -- whole sequences: fixed length ``[B, T, ...]`` or packed
  ``[1, T, ...]`` with ``cu_seqlens``, fp32 states in and out, differentiable.
* :func:`selective_scan_step` -- one token per sequence on a pool of fp32 states
  that is updated in place (serving).

The work is ``gdn2_selective_fwd`` / ``gdn2_selective_bwd`` / ``gdn2_selective_step``
of ``libgdn2_b200.so``; there is no CPU path.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from .. import _native as N
from .gated_scan import _rows

__all__ = ["SelectiveScanFunction", "selective_scan", "selective_scan_step"]

MAX_STATES = 64


def _f32(p):
    """A parameter as the kernels read it (its address is all that is used)."""
    if p is None or p.dtype is torch.float32 and p.is_contiguous():
        return p
    return p.detach().float().contiguous()


class _Call:
    """Sizes, packing, row strides and parameters of one call."""

    def __init__(self, x, dt, A, B, C, D, z, dt_bias, softplus, cu, lead):
        b, t = (x.shape[0], 1) if lead == 1 else x.shape[:2]
        d, n = A.shape
        g = 1 if B.ndim == lead + 1 else B.shape[lead]
        self.b, self.t, self.d, self.g, self.states = b, t, d, g, n
        self.softplus, self.cu = softplus, cu
        self.n = b if cu is None else cu.numel() - 1
        self.x, self.ldx = _rows(x, b, t, d)
        self.dt, self.lddt = _rows(dt, b, t, d)
        self.z, self.ldz = (None, d) if z is None else _rows(z, b, t, d)
        self.B, self.ldb = _rows(B, b, t, g * n)
        self.C, self.ldc = _rows(C, b, t, g * n)
        self.A, self.D, self.bias = _f32(A), _f32(D), _f32(dt_bias)

    def problem(self, lddy=None):
        return N.SelectiveProblem(self.b, self.d, self.g, self.states, self.t, N.dtype_code(self.x.dtype),
                                  N.dtype_code(self.dt.dtype), int(self.softplus), self.n, N.addr(self.cu),
                                  self.ldx, self.lddt, self.ldz, self.ldb, self.ldc, lddy or self.d)

    def inputs(self):
        return [N.addr(p) for p in (self.x, self.dt, self.A, self.B, self.C, self.D, self.z, self.bias)]


def _workspace(prob, backward, device):
    size = N.load().gdn2_selective_workspace_bytes(prob, backward)
    return (torch.empty(size, dtype=torch.uint8, device=device) if size else None), size


def _forward(call, shape, h0, want_final, keep):
    lib, dev = N.load(), call.x.device
    prob = call.problem()
    y = torch.empty(shape, dtype=call.x.dtype, device=dev)
    ht = torch.empty(call.n, call.d, call.states, dtype=torch.float32, device=dev) if want_final else None
    saved = None
    if keep:
        saved = torch.empty(lib.gdn2_selective_saved_bytes(prob) // 4, dtype=torch.float32, device=dev)
    with N.on_device(dev.index):
        ws, size = _workspace(prob, 0, dev)
        N.check(lib.gdn2_selective_fwd(prob, *call.inputs(), N.addr(h0), N.addr(y), N.addr(ht),
                                       N.addr(saved), N.addr(ws), size, N.raw_stream(dev.index)),
                "gdn2_selective_fwd")
    return y, ht, saved


class SelectiveScanFunction(torch.autograd.Function):
    """y, ht of :func:`selective_scan` with gradients for every tensor."""

    @staticmethod
    def forward(ctx, x, dt, A, B, C, D, z, dt_bias, h0, softplus, cu, want_final):
        call = _Call(x, dt, A, B, C, D, z, dt_bias, softplus, cu, 2)
        y, ht, saved = _forward(call, x.shape, h0, want_final, keep=True)
        ctx.save_for_backward(x, dt, A, B, C, D, z, dt_bias, h0, cu, saved)
        ctx.softplus = softplus
        ctx.set_materialize_grads(False)
        return y, ht

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dht):
        x, dt, A, B, C, D, z, dt_bias, h0, cu, saved = ctx.saved_tensors
        if dy is None and dht is None:
            return (None,) * 12
        lib, dev = N.load(), x.device
        call = _Call(x, dt, A, B, C, D, z, dt_bias, ctx.softplus, cu, 2)
        dy = torch.zeros_like(x) if dy is None else dy.to(x.dtype)
        dy, lddy = _rows(dy, call.b, call.t, call.d)
        dht = dht.float().contiguous() if dht is not None else None
        prob = call.problem(lddy)
        new = lambda p: None if p is None else torch.empty(p.shape, dtype=p.dtype, device=dev)
        wide = lambda p: None if p is None else torch.empty(p.shape, dtype=torch.float32, device=dev)
        dx, ddt, dB, dC, dz = map(new, (x, dt, B, C, z))
        dA, dD, dbias, dh0 = map(wide, (A, D, dt_bias, h0))
        with N.on_device(dev.index):
            ws, size = _workspace(prob, 1, dev)
            N.check(lib.gdn2_selective_bwd(
                prob, *call.inputs(), N.addr(h0), N.addr(saved), N.addr(dy), N.addr(dht), N.addr(dx),
                N.addr(ddt), N.addr(dA), N.addr(dB), N.addr(dC), N.addr(dD), N.addr(dz), N.addr(dbias),
                N.addr(dh0), N.addr(ws), size, N.raw_stream(dev.index)), "gdn2_selective_bwd")
        like = lambda g, p: None if p is None else g.to(p.dtype)
        return (dx, ddt, like(dA, A), dB, dC, like(dD, D), dz, like(dbias, dt_bias), dh0, None, None, None)


def _check(fn, x, dt, A, B, C, D, z, dt_bias, lead):
    device, dtype = x.device, x.dtype
    for t in (x, dt, A, B, C, D, z, dt_bias):
        if t is not None and not t.is_cuda:
            raise RuntimeError(f"{fn}: inputs must be CUDA tensors -- the B200 build has no CPU path")
    if x.ndim != lead + 1 or x.shape[-1] == 0:
        raise ValueError(f"{fn}: x must be {'[B, T, D]' if lead == 2 else '[N, D]'}; got {tuple(x.shape)}")
    d = x.shape[-1]
    if A.ndim != 2 or A.shape[0] != d or A.shape[1] == 0:
        raise ValueError(f"{fn}: A must be [{d}, states]; got {tuple(A.shape)}")
    n = A.shape[1]
    if n > MAX_STATES:
        raise NotImplementedError(f"{fn}: up to {MAX_STATES} states are supported; got {n}")
    for name, t in (("dt", dt), ("z", z)):
        if t is not None and t.shape != x.shape:
            raise ValueError(f"{fn}: {name} must have x's shape {tuple(x.shape)}; got {tuple(t.shape)}")
    if B.shape != C.shape or B.ndim not in (lead + 1, lead + 2) or B.shape[:lead] != x.shape[:lead] \
            or B.shape[-1] != n:
        raise ValueError(f"{fn}: B and C must be {list(x.shape[:lead])} + [{n}] or [groups, {n}]; got "
                         f"{tuple(B.shape)} and {tuple(C.shape)}")
    if B.ndim == lead + 2 and (B.shape[lead] == 0 or d % B.shape[lead]):
        raise ValueError(f"{fn}: {d} channels do not divide into {B.shape[lead]} groups")
    for name, t in (("D", D), ("dt_bias", dt_bias)):
        if t is not None and t.shape != (d,):
            raise ValueError(f"{fn}: {name} must be [{d}]; got {tuple(t.shape)}")
    for name, t in (("dt", dt), ("A", A), ("B", B), ("C", C), ("D", D), ("z", z), ("dt_bias", dt_bias)):
        if t is None:
            continue
        if t.device != device:
            raise ValueError(f"{fn}: {name} is on {t.device}, x on {device}")
        if t.dtype is not torch.float32:
            N.dtype_code(t.dtype)
    N.dtype_code(dtype)
    for name, t in (("B", B), ("C", C), ("z", z)):
        if t is not None and t.dtype is not dtype:
            raise NotImplementedError(f"{fn}: x ({dtype}) and {name} ({t.dtype}) must share a dtype")
    if dt.dtype != x.dtype and dt.dtype != torch.float32:
        raise NotImplementedError(f"{fn}: dt ({dt.dtype}) must be float32 or x's dtype ({x.dtype})")


def selective_scan(
    x: torch.Tensor,
    dt: torch.Tensor,
    A: torch.Tensor,
    B: torch.Tensor,
    C: torch.Tensor,
    D: torch.Tensor | None = None,
    z: torch.Tensor | None = None,
    *,
    dt_bias: torch.Tensor | None = None,
    dt_softplus: bool = False,
    initial_state: torch.Tensor | None = None,
    output_final_state: bool = False,
    cu_seqlens: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    r"""``h_t = exp(d_t A) h_{t-1} + d_t x_t B_t``, ``y_t = (sum_n h_t C_t + D x_t) silu(z_t)``
    over the second dimension, with ``d = softplus(dt + dt_bias)`` (without
    ``dt_softplus``, ``dt + dt_bias``).

    x: ``[B, T, D]`` (float32, bfloat16 or float16); dt: x's shape in float32 or x's
    dtype; A: ``[D, N]``, N up to 64 (negative where states decay); B, C:
    ``[B, T, N]``, or ``[B, T, G, N]`` for G groups of D / G neighbouring channels; D
    and dt_bias: ``[D]`` or None; z: x's shape, or None for no gate.  A, D and dt_bias
    are taken in float32.  ``initial_state`` and the returned final state (None unless
    ``output_final_state``) are float32 ``[n, D, N]``.  With ``cu_seqlens`` (``[n+1]``,
    from 0 to T, not decreasing; not checked on the device) B must be 1 and the n
    packed sequences, empty ones included, each start from their own state; n = B
    otherwise.  Returns ``(y, final_state)``, y in x's dtype; states and sums are
    float32.  Differentiable (once, in reverse mode) in every tensor but
    ``cu_seqlens``; for that the forward keeps a state every 16 tokens, ``D N / 4``
    bytes a token (N rounded up to 4), and the backward takes ``8 N`` bytes of scratch a
    token for each tile of 64, 32, 16 or 8 channels (up to 8, 16, 32 or 64 states): half
    of what is kept, as much, twice or four times as much, and more where groups do not
    fill their tiles, since each group has tiles of its own.  The factor
    by which states grow (``d A > 0``) must stay finite over a chunk of the time axis.
    Rows may be strided (slices of a fused projection).
    """
    fn = "selective_scan"
    _check(fn, x, dt, A, B, C, D, z, dt_bias, 2)
    n = x.shape[0]
    cu = None
    if cu_seqlens is not None:
        if x.shape[0] != 1:
            raise ValueError(
                f"The batch size is expected to be 1 rather than {x.shape[0]} when using "
                "`cu_seqlens`. Please flatten variable-length inputs before processing.")
        if cu_seqlens.ndim != 1 or cu_seqlens.numel() < 1 or cu_seqlens.is_floating_point():
            raise ValueError("cu_seqlens must be a 1-D tensor of offsets")
        n = cu_seqlens.numel() - 1
    if n > N.INT32_MAX:
        raise ValueError(f"{fn}: up to 2^31 - 1 sequences are supported; got {n}")
    if cu_seqlens is not None:
        cu = cu_seqlens.to(device=x.device, dtype=torch.int32).contiguous()
    h0 = initial_state
    if h0 is not None:
        if h0.dtype != torch.float32:
            raise TypeError("initial_state must be in float32.")
        if h0.device != x.device or tuple(h0.shape) != (n, *A.shape):
            raise ValueError(f"initial_state must be [{n}, {A.shape[0]}, {A.shape[1]}] on {x.device}; "
                             f"got {tuple(h0.shape)} on {h0.device}")
        h0 = h0.contiguous()
    leaves = (x, dt, A, B, C, D, z, dt_bias, h0)
    if N.forward_mode(*leaves) or torch.is_grad_enabled() and any(
            t is not None and t.requires_grad for t in leaves):
        return SelectiveScanFunction.apply(*leaves, bool(dt_softplus), cu, bool(output_final_state))
    call = _Call(x, dt, A, B, C, D, z, dt_bias, bool(dt_softplus), cu, 2)
    y, ht, _ = _forward(call, x.shape, h0, bool(output_final_state), keep=False)
    return y, ht


@torch.no_grad()
def selective_scan_step(
    x: torch.Tensor,
    dt: torch.Tensor,
    A: torch.Tensor,
    B: torch.Tensor,
    C: torch.Tensor,
    D: torch.Tensor | None = None,
    z: torch.Tensor | None = None,
    *,
    dt_bias: torch.Tensor | None = None,
    dt_softplus: bool = False,
    state: torch.Tensor,
    state_indices: torch.Tensor | None = None,
) -> torch.Tensor:
    r"""One token for each of n sequences (inference only).

    Inputs as in :func:`selective_scan` without the time dimension (x ``[n, D]``, B
    and C ``[n, N]`` or ``[n, G, N]``).  ``state``: float32 pool ``[S, D, N]``, updated
    in place; sequence i uses row ``state_indices[i]`` (row i without indices).  An
    index outside ``[0, S)`` marks padding: no state changes and its row of y is
    zero.  Two sequences must not name the same row.  Returns y ``[n, D]`` in x's
    dtype.
    """
    fn = "selective_scan_step"
    _check(fn, x, dt, A, B, C, D, z, dt_bias, 1)
    n, per = x.shape[0], A.shape[0] * A.shape[1]
    if state.dtype != torch.float32:
        raise TypeError("state must be in float32.")
    if state.device != x.device or state.shape[1:] != A.shape:
        raise ValueError(f"state must be [S, {A.shape[0]}, {A.shape[1]}] on {x.device}; got "
                         f"{tuple(state.shape)} on {state.device}")
    if n > N.INT32_MAX or state.shape[0] > N.INT32_MAX:
        raise ValueError(f"{fn}: up to 2^31 - 1 sequences and states are supported; got {n} and "
                         f"{state.shape[0]}")
    if not state.is_contiguous() and (not state[:1].is_contiguous() or (
            state.shape[0] > 1 and state.stride(0) < per)):
        raise ValueError("state must hold each sequence's channels contiguously")
    idx = None
    if state_indices is not None:
        if state_indices.shape != (n,) or state_indices.is_floating_point():
            raise ValueError(f"state_indices must be {n} integers; got "
                             f"{tuple(state_indices.shape)} {state_indices.dtype}")
        idx = state_indices
        if idx.dtype is not torch.int32:  # outside the pool stays outside in 32 bits
            idx = idx.to(torch.int64).clamp(-1, state.shape[0]).to(torch.int32)
        if idx.device != x.device or not idx.is_contiguous():
            idx = idx.to(x.device).contiguous()
    elif state.shape[0] < n:
        raise ValueError(f"{n} sequences need as many states; got {state.shape[0]}")
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if n == 0:
        return y
    if state.shape[0] == 0:
        return y.zero_()
    call = _Call(x, dt, A, B, C, D, z, dt_bias, bool(dt_softplus), None, 1)
    index = x.device.index
    with N.on_device(index):
        N.check(N.load().gdn2_selective_step(
            call.problem(), *call.inputs(), N.addr(state), max(state.stride(0), per), state.shape[0],
            N.addr(idx), N.addr(y), N.raw_stream(index)), "gdn2_selective_step")
    increment_version(state)  # autograd does not see the kernel's writes
    return y
