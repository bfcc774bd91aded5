"""The norm of many gradients and its clipping on B200.

* :func:`grad_norm` -- the norm of a list of tensors taken together, with the
  coefficient that clips it, all left on the device: what
  :class:`~qwendopamine_b200.AdamW` takes as ``grad_scale`` and ``found_inf``,
  so that clipping costs one read of the gradients;
* :func:`clip_grad_norm_` -- the same, and the gradients scaled in place.

The work is ``gdn2_grad_norm`` and ``gdn2_grad_scale`` of ``libgdn2_b200.so``
(256 tensors a launch); there is no CPU path.
"""

from __future__ import annotations

import math
import struct
from itertools import chain
from operator import attrgetter
from typing import NamedTuple

import torch
from torch.autograd.graph import increment_version

from .. import _native as N

__all__ = ["GradNorm", "clip_grad_norm_", "grad_norm"]

_ptr, _numel, _dense = torch.Tensor.data_ptr, torch.Tensor.numel, torch.Tensor.is_contiguous
_dtype, _device = attrgetter("dtype"), torch.Tensor.get_device


class GradNorm(NamedTuple):
    """Results of :func:`grad_norm`: float32 scalars on the gradients' device."""

    norm: torch.Tensor
    clip_coef: torch.Tensor
    found_inf: torch.Tensor


def _norm_code(fn, norm_type):
    if norm_type == 2:
        return 2
    if norm_type == math.inf:
        return 0
    raise ValueError(f"{fn}: norm_type must be 2 or inf; got {norm_type}")


def _one_list(fn, tensors):
    if isinstance(tensors, torch.Tensor):
        tensors = [tensors]
    tensors = list(tensors)
    if not tensors:
        raise ValueError(f"{fn}: needs at least one tensor")
    device = tensors[0].device
    if device.type != "cuda":
        raise RuntimeError(f"{fn}: tensors must be CUDA tensors -- the B200 build has no CPU path")
    if set(map(_device, tensors)) != {device.index}:
        raise ValueError(f"{fn}: tensors must all be on {device}")
    if any(t.layout is not torch.strided for t in tensors):
        raise RuntimeError(f"{fn} (B200 build) does not take sparse gradients")
    return tensors, device


def _table(tensors):
    """gdn2_grad_tensor rows: address, number of elements, dtype."""
    codes = {dt: N.dtype_code(dt) for dt in set(map(_dtype, tensors))}
    rows = zip(map(_ptr, tensors), map(_numel, tensors), (codes[t.dtype] for t in tensors))
    return struct.pack(f"{3 * len(tensors)}q", *chain.from_iterable(rows))


def _measure(table, n, device, kind, max_norm):
    lib = N.load()
    out = torch.empty(3, dtype=torch.float32, device=device)
    size = lib.gdn2_grad_norm_workspace_bytes(n)
    ws = torch.empty(size, dtype=torch.uint8, device=device)
    prob = N.GradProblem(kind, -1.0 if max_norm is None else max_norm)
    N.check(lib.gdn2_grad_norm(prob, table, n, out.data_ptr(), ws.data_ptr(), size,
                               N.raw_stream(device.index)), "gdn2_grad_norm")
    return GradNorm(*out.unbind())


def _limit(fn, max_norm):
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError(f"{fn}: max_norm must not be negative; got {max_norm}")
    return max_norm


@torch.no_grad()
def grad_norm(
    grads: torch.Tensor | list[torch.Tensor],
    *,
    max_norm: float | None = None,
    norm_type: float = 2.0,
) -> GradNorm:
    r"""Norm of ``grads`` taken as one vector, left on the device.

    grads: CUDA tensors in float32, bfloat16 or float16, mixed as they come, all
    on one device.  ``norm_type``: 2, or ``math.inf`` for the largest magnitude.
    Returns float32 scalars: ``norm``; ``clip_coef``, ``min(1, max_norm / (norm +
    1e-6))`` (1 without ``max_norm``, and where the norm is not finite); and
    ``found_inf``, 1 where the norm is not finite, else 0.  ``AdamW.step`` takes
    the last two as ``grad_scale`` and ``found_inf``.  A tensor that is listed
    twice counts twice; the norm of nothing but empty tensors is 0.  Squares are added
    in float32 up to 64 at a time (in float64 where float32 does not hold their sum)
    and those sums in float64.  Equal inputs give equal bits.
    """
    kind = _norm_code("grad_norm", norm_type)
    if max_norm is not None:
        max_norm = _limit("grad_norm", max_norm)
    grads, device = _one_list("grad_norm", grads)
    if not all(map(_dense, grads)):
        grads = [g.contiguous() for g in grads]
    with N.on_device(device.index):
        return _measure(_table(grads), len(grads), device, kind, max_norm)


@torch.no_grad()
def clip_grad_norm_(
    grads: torch.Tensor | list[torch.Tensor],
    max_norm: float,
    *,
    norm_type: float = 2.0,
) -> GradNorm:
    r"""As :func:`grad_norm`, and ``grads`` multiplied in place by ``clip_coef``.

    What is scaled is what is given, ``[p.grad for p in model.parameters()]``: unlike
    the function of this name in ``torch.nn.utils`` it takes gradients, and refuses
    ``nn.Parameter``.  Each value is multiplied in float32 and rounded once to its
    tensor's dtype.  Gradients whose norm is 1e-6 and more within ``max_norm``, or not
    finite, stay as they are.
    The tensors must fill their memory without gaps and must not overlap one
    another.  What is scaled counts as changed in place for autograd, also where
    the coefficient turns out to be 1 (nothing is read on the host).
    """
    fn = "clip_grad_norm_"
    kind, max_norm = _norm_code(fn, norm_type), _limit(fn, max_norm)
    grads = [grads] if isinstance(grads, torch.Tensor) else list(grads)
    if any(isinstance(g, torch.nn.Parameter) for g in grads):
        raise TypeError(f"{fn}: takes gradients, and scales what it is given; got parameters "
                        "(pass [p.grad for p in model.parameters()])")
    grads, device = _one_list(fn, grads)
    for g in grads:  # the order of the elements does not matter, gaps do
        if not g.is_contiguous() and not torch.ops.aten.is_non_overlapping_and_dense(g):
            raise ValueError(f"{fn}: each tensor must fill its memory without gaps; got strides "
                             f"{g.stride()} for {tuple(g.shape)}")
    table, n = _table(grads), len(grads)
    with N.on_device(device.index):
        r = _measure(table, n, device, kind, max_norm)
        N.check(N.load().gdn2_grad_scale(table, n, r.clip_coef.data_ptr(),
                                         N.raw_stream(device.index)), "gdn2_grad_scale")
    increment_version(grads)  # autograd does not see the kernel's writes
    return r
