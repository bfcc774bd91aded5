"""Log probabilities of given tokens on B200, with entropy, the most likely
alternatives and the logits' gradient.

:func:`token_logprobs` is a decoder's loss (``-logprobs`` of the targets, an
entropy bonus) and what a serving loop reports for the tokens it chose.  The
forward reads the logits once and keeps four numbers per row; the backward
reads them again and writes the gradient.  The work is one launch each of
``gdn2_logprob_fwd`` / ``gdn2_logprob_bwd`` from ``libgdn2_b200.so``; there is
no CPU path.
"""

from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from .. import _native as N

__all__ = ["TokenLogprobs", "TokenLogprobsFunction", "token_logprobs"]


class TokenLogprobs(NamedTuple):
    """Results of :func:`token_logprobs` (None for what was not asked for)."""

    logprobs: torch.Tensor
    entropy: torch.Tensor | None
    top_logprobs: torch.Tensor | None
    top_ids: torch.Tensor | None


def _matrix(logits):
    """``logits`` as ``[rows, V]`` with one row stride, copied only if need be."""
    V = logits.shape[-1]
    if logits.ndim == 2 and logits.is_contiguous():
        return logits, V
    x = logits.reshape(-1, V)
    if (x.stride(1) != 1 and V > 1) or (x.shape[0] > 1 and x.stride(0) < V):
        x = x.contiguous()
    return x, max(x.stride(0), V)


def _problem(x, ld, top_k, temperature, ignore_index):
    return N.LogprobProblem(x.shape[0], ld, ignore_index, x.shape[1], N.dtype_code(x.dtype), top_k,
                            temperature)


def _forward(x, ld, ids, top_k, entropy, temperature, ignore_index, keep):
    rows, dev = x.shape[0], x.device
    f32 = lambda *s: torch.empty(s, dtype=torch.float32, device=dev)
    logp = f32(rows)
    ent = f32(rows) if entropy else None
    top = f32(rows, top_k) if top_k else None
    top_ids = torch.empty(rows, top_k, dtype=torch.int64, device=dev) if top_k else None
    stats = f32(rows, 4) if keep else None
    with N.on_device(dev.index):
        N.check(N.load().gdn2_logprob_fwd(
            _problem(x, ld, top_k, temperature, ignore_index), N.addr(x), N.addr(ids), N.addr(logp),
            N.addr(ent), N.addr(top), N.addr(top_ids), N.addr(stats), N.raw_stream(dev.index)),
            "gdn2_logprob_fwd")
    return logp, ent, top, top_ids, stats


class TokenLogprobsFunction(torch.autograd.Function):
    """(logprobs, entropy, top_logprobs, top_ids) of rows of logits; the first
    two are differentiable."""

    @staticmethod
    def forward(ctx, logits, ids, top_k, entropy, temperature, ignore_index):
        x, ld = _matrix(logits)
        logp, ent, top, top_ids, stats = _forward(x, ld, ids, top_k, entropy, temperature,
                                                  ignore_index, keep=True)
        ctx.save_for_backward(logits, ids, stats)
        ctx.meta = (temperature, ignore_index)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(*(t for t in (top, top_ids) if t is not None))
        return logp, ent, top, top_ids

    @staticmethod
    @once_differentiable
    def backward(ctx, dlogp, dent, dtop, dtop_ids):
        logits, ids, stats = ctx.saved_tensors
        if dlogp is None and dent is None:
            return None, None, None, None, None, None
        temperature, ignore_index = ctx.meta
        x, ld = _matrix(logits)
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        dlogp = dlogp.float().contiguous() if dlogp is not None else None
        dent = dent.float().contiguous() if dent is not None else None
        with N.on_device(x.device.index):
            N.check(N.load().gdn2_logprob_bwd(
                _problem(x, ld, 0, temperature, ignore_index), N.addr(x), N.addr(ids), N.addr(stats),
                N.addr(dlogp), N.addr(dent), N.addr(dx), N.raw_stream(x.device.index)),
                "gdn2_logprob_bwd")
        return dx.view(logits.shape), None, None, None, None, None


def token_logprobs(
    logits: torch.Tensor,
    token_ids: torch.Tensor,
    *,
    top_k: int = 0,
    entropy: bool = False,
    temperature: float = 1.0,
    ignore_index: int = -100,
) -> TokenLogprobs:
    r"""Log probability of ``token_ids`` under ``softmax(logits / temperature)``.

    logits: ``[..., V]`` in float32, bfloat16 or float16 (rows may be strided);
    token_ids: ``[...]`` integers.  Returns float32 ``logprobs`` ``[...]``;
    with ``entropy`` also the rows' entropies in nats; with ``top_k`` (at most
    128) the ``top_k`` largest log probabilities ``[..., top_k]`` in falling
    order and their int64 ids, equal ones by rising id.  Sums are float32
    whatever the logits' type.

    -inf logits (a mask) have probability zero; a row of only -inf has log
    probability -inf, entropy 0 and no gradient.  Rows whose id is
    ``ignore_index`` give 0 and 0 (-inf and id -1 as alternatives), no
    gradient, and are not read; an id outside the vocabulary gives NaN.  NaN
    logits make the row's results NaN and come last among the alternatives.
    Differentiable (once, in reverse mode) in ``logits`` through ``logprobs``
    and ``entropy``.
    """
    if not logits.is_cuda:
        raise RuntimeError("token_logprobs: logits must be a CUDA tensor -- the B200 build has no "
                           "CPU path")
    if logits.ndim < 1 or not 1 <= logits.shape[-1] <= N.INT32_MAX:
        raise ValueError(f"token_logprobs: logits need a vocabulary of up to 2^31 - 1 tokens; got "
                         f"{tuple(logits.shape)}")
    if token_ids.shape != logits.shape[:-1] or token_ids.is_floating_point() \
            or token_ids.dtype == torch.bool:
        raise ValueError(f"token_logprobs: token_ids must be {tuple(logits.shape[:-1])} integers; "
                         f"got {tuple(token_ids.shape)} {token_ids.dtype}")
    if not 0 <= top_k <= logits.shape[-1]:
        raise ValueError(f"token_logprobs: top_k must be in 0 .. {logits.shape[-1]}; got {top_k}")
    N.dtype_code(logits.dtype)
    lead = logits.shape[:-1]
    ids = token_ids.to(device=logits.device, dtype=torch.int64).reshape(-1).contiguous()
    args = (int(top_k), bool(entropy), float(temperature), int(ignore_index))
    if logits.requires_grad and torch.is_grad_enabled() or N.forward_mode(logits):
        logp, ent, top, top_ids = TokenLogprobsFunction.apply(logits, ids, *args)
    else:
        logp, ent, top, top_ids, _ = _forward(*_matrix(logits), ids, *args, keep=False)
    if len(lead) == 1:
        return TokenLogprobs(logp, ent, top, top_ids)
    shaped = lambda t, *more: None if t is None else t.view((*lead, *more))
    return TokenLogprobs(shaped(logp), shaped(ent), shaped(top, top_k), shaped(top_ids, top_k))
