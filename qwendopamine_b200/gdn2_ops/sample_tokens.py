"""The next token of each sequence on B200, from logits and given random numbers.

:func:`sample_tokens` is the step of a serving loop between the model's logits
and :func:`~qwendopamine_b200.token_logprobs` of the token that was chosen:
temperature, top-k, top-p and min-p, the same for all rows or each row its own.
One launch of ``gdn2_sample`` from ``libgdn2_b200.so``; there is no CPU path.
"""

from __future__ import annotations

import math

import torch

from .. import _native as N
from .token_logprobs import _matrix

__all__ = ["sample_tokens"]


def _option(name, value, lead, device, dtype, low, high):
    """A number (checked) or a tensor of one value for each row: (number, tensor)."""
    if isinstance(value, torch.Tensor):
        if value.shape != lead:
            raise ValueError(f"sample_tokens: {name} must be a number or {tuple(lead)} of them; got "
                             f"{tuple(value.shape)}")
        if value.is_floating_point() != dtype.is_floating_point or value.dtype == torch.bool:
            raise ValueError(f"sample_tokens: {name} must be "
                             f"{'floating-point' if dtype.is_floating_point else 'whole'} numbers; "
                             f"got {value.dtype}")
        if dtype is torch.int32 and value.dtype is torch.int64:
            value = value.clamp(0, N.INT32_MAX)  # what is larger than a vocabulary keeps all of it
        if value.dtype is not dtype or value.device != device or not value.is_contiguous():
            value = value.to(device, dtype).contiguous()
        return 0, value
    if not low <= value <= high:
        raise ValueError(f"sample_tokens: {name} must be in {low} .. {high}; got {value}")
    return value, None


@torch.no_grad()
def sample_tokens(
    logits: torch.Tensor,
    uniform: torch.Tensor,
    *,
    temperature: float | torch.Tensor = 1.0,
    top_k: int | torch.Tensor = 0,
    top_p: float | torch.Tensor = 1.0,
    min_p: float | torch.Tensor = 0.0,
) -> torch.Tensor:
    r"""One token id for each row of ``logits``, int64 ``[...]``.

    logits: ``[..., V]`` in float32, bfloat16 or float16 (rows may be strided);
    uniform: ``[...]`` float32, a random number in [0, 1) for each row
    (``torch.rand``): the same numbers give the same tokens.  ``temperature``,
    ``top_k``, ``top_p`` and ``min_p`` are numbers or tensors ``[...]``, one value
    for each row.

    With ``w = exp((logits - max) / temperature)``: ``min_p`` keeps ``w >= min_p``;
    of those ``top_k`` keeps the k largest; of those ``top_p`` keeps, in falling
    order, up to the first whose running sum reaches ``top_p`` of their sum
    (equal logits rank by rising id).  The token is the lowest id whose running
    sum of kept weights, by rising id, exceeds ``uniform`` times their sum.
    Weights and sums are float64 (weights below 2^-1022 are zero); -0 and 0 are equal.

    ``temperature`` 0, ``top_k`` 1 and ``top_p`` 0 take the first maximum;
    ``top_k`` 0, ``top_p`` 1 and ``min_p`` 0 keep everything.  In tensors, which
    are not checked on the host, values below those count as them, and above 1 as
    1.  -inf logits (a mask) are never taken.  A row without a distribution -- NaN
    or +inf among its logits, all of them -inf, or NaN in its uniform or options --
    gives -1.  Not differentiable.
    """
    if not logits.is_cuda:
        raise RuntimeError("sample_tokens: logits must be a CUDA tensor -- the B200 build has no "
                           "CPU path")
    if logits.ndim < 1 or not 1 <= logits.shape[-1] <= N.INT32_MAX:
        raise ValueError(f"sample_tokens: logits need a vocabulary of up to 2^31 - 1 tokens; got "
                         f"{tuple(logits.shape)}")
    code, lead, device = N.dtype_code(logits.dtype), logits.shape[:-1], logits.device
    if uniform.shape != lead or uniform.dtype != torch.float32 or uniform.device != device:
        raise ValueError(f"sample_tokens: uniform must be {tuple(lead)} float32 on {device}; got "
                         f"{tuple(uniform.shape)} {uniform.dtype} on {uniform.device}")
    f32 = torch.float32
    t, t_rows = _option("temperature", temperature, lead, device, f32, 0, 1.7e308)
    k, k_rows = _option("top_k", top_k, lead, device, torch.int32, 0, math.inf)
    p, p_rows = _option("top_p", top_p, lead, device, f32, 0, 1)
    q, q_rows = _option("min_p", min_p, lead, device, f32, 0, 1)
    x, ld = _matrix(logits)
    uniform = uniform.contiguous()
    ids = torch.empty(lead, dtype=torch.int64, device=device)
    prob = N.SampleProblem(x.shape[0], ld, x.shape[1], code, int(min(k, x.shape[1])), t, p, q)
    with N.on_device(device.index):
        N.check(N.load().gdn2_sample(prob, N.addr(x), N.addr(uniform), N.addr(t_rows), N.addr(k_rows),
                                     N.addr(p_rows), N.addr(q_rows), N.addr(ids),
                                     N.raw_stream(device.index)), "gdn2_sample")
    return ids
