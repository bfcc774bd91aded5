"""AdamW on B200: one launch for many tensors, states in 32 or 8 bits.

* :func:`adamw_step` -- one step on lists of tensors (``gdn2_adamw_step`` of
  ``libgdn2_b200.so``; there is no CPU path);
* :class:`AdamW` -- the ``torch.optim.Optimizer`` around it.

8-bit states are ``torch.float8_e4m3fn`` codes with one float32 scale for each
256 consecutive elements of a tensor: the first moment is ``code * scale``, the
second moment ``(code * scale) ** 2`` (its root is what is held), and all zeros
is the state before the first step.
"""

from __future__ import annotations

import math
import struct
from itertools import chain
from operator import attrgetter

import torch
from torch.autograd.graph import increment_version

from .. import _native as N

__all__ = ["AdamW", "adamw_step", "STATE_BLOCK"]

STATE_BLOCK = 256  # elements that share a scale in the 8-bit states

_ptr, _numel, _dense = torch.Tensor.data_ptr, torch.Tensor.numel, torch.Tensor.is_contiguous
_dtype, _device = attrgetter("dtype"), torch.Tensor.get_device


# places of the lists in a row of gdn2_adamw_tensor words
_COLUMN = {"params": 0, "grads": 1, "exp_avgs": 2, "exp_avg_sqs": 3, "exp_avg_scales": 4,
           "exp_avg_sq_scales": 5, "master_params": 6}


def _scalar(name, t, device):
    if t is None:
        return None
    if t.numel() != 1 or t.dtype != torch.float32 or t.device != device:
        raise ValueError(f"adamw_step: {name} must be one float32 value on {device}")
    return t


def adamw_step(
    params: list[torch.Tensor],
    grads: list[torch.Tensor],
    exp_avgs: list[torch.Tensor],
    exp_avg_sqs: list[torch.Tensor],
    *,
    step: int,
    lr: float,
    betas: tuple[float, float] = (0.9, 0.999),
    eps: float = 1e-8,
    weight_decay: float = 1e-2,
    exp_avg_scales: list[torch.Tensor] | None = None,
    exp_avg_sq_scales: list[torch.Tensor] | None = None,
    master_params: list[torch.Tensor] | None = None,
    grad_scale: torch.Tensor | None = None,
    found_inf: torch.Tensor | None = None,
) -> None:
    r"""One AdamW step, in place, on parallel lists of contiguous CUDA tensors.

    ``params`` share one dtype (float32, bfloat16, float16); ``grads`` have it
    or are all float32.  ``exp_avgs`` / ``exp_avg_sqs`` are float32, or
    ``float8_e4m3fn`` codes with ``exp_avg_scales`` / ``exp_avg_sq_scales``
    (float32, ``ceil(numel / 256)`` each).  With ``master_params`` (float32)
    the step is taken on those and ``params`` receive their rounding; without,
    16-bit parameters are rounded to nearest after the step.  ``step`` counts
    from 1.  ``grad_scale`` (a float32 device scalar) multiplies the gradients,
    and a nonzero ``found_inf`` leaves everything as it is; neither is read on
    the host.  A captured call keeps ``step`` and ``lr``.  What is written counts as changed in place for autograd.
    """
    n = len(params)
    lists = {"params": params, "grads": grads, "exp_avgs": exp_avgs, "exp_avg_sqs": exp_avg_sqs}
    if (exp_avg_scales is None) != (exp_avg_sq_scales is None):
        raise ValueError("adamw_step: 8-bit states need both lists of scales")
    eight = exp_avg_scales is not None
    if eight:
        lists.update(exp_avg_scales=exp_avg_scales, exp_avg_sq_scales=exp_avg_sq_scales)
    if master_params is not None:
        lists["master_params"] = master_params
    for name, x in lists.items():
        if len(x) != n:
            raise ValueError(f"adamw_step: {name} has {len(x)} tensors, params {n}")
    if n == 0:
        return
    device, dtype, gdtype = params[0].device, params[0].dtype, grads[0].dtype
    if device.type != "cuda":
        raise RuntimeError("adamw_step: tensors must be CUDA tensors -- the B200 build has no CPU "
                           "path")
    code = N.dtype_code(dtype)
    if gdtype != dtype and gdtype != torch.float32:
        raise NotImplementedError(f"adamw_step: gradients ({gdtype}) must be float32 or have the "
                                  f"parameters' dtype ({dtype})")
    sdtype = torch.float8_e4m3fn if eight else torch.float32
    want = {"params": dtype, "grads": gdtype, "exp_avgs": sdtype, "exp_avg_sqs": sdtype}
    sizes = list(map(_numel, params))
    # one row of 64-bit words for each tensor, filled a column (a list) at a time
    words = [0] * (n * N.ADAMW_TENSOR_WORDS)
    words[N.ADAMW_TENSOR_WORDS - 1::N.ADAMW_TENSOR_WORDS] = sizes
    for name, x in lists.items():
        if set(map(_dtype, x)) != {want.get(name, torch.float32)} \
                or set(map(_device, x)) != {device.index}:
            raise ValueError(f"adamw_step: {name} must all be {want.get(name, torch.float32)} on "
                             f"{device}")
        if not all(map(_dense, x)):
            if x is not grads:
                raise ValueError(f"adamw_step: {name} must be contiguous")
            x = grads = [g.contiguous() for g in grads]
        if name.endswith("scales"):
            if list(map(_numel, x)) != [-(-s // STATE_BLOCK) for s in sizes]:
                raise ValueError(f"adamw_step: {name} need one value for each {STATE_BLOCK} "
                                 "elements")
        elif x is not params and list(map(_numel, x)) != sizes:
            raise ValueError(f"adamw_step: {name} must have the parameters' sizes")
        words[_COLUMN[name]::N.ADAMW_TENSOR_WORDS] = list(map(_ptr, x))
    prob = N.AdamWProblem(code, N.dtype_code(gdtype), 8 if eight else 32, int(step), lr, betas[0],
                          betas[1], eps, weight_decay,
                          N.addr(_scalar("grad_scale", grad_scale, device)),
                          N.addr(_scalar("found_inf", found_inf, device)))
    with N.on_device(device.index):
        N.check(N.load().gdn2_adamw_step(prob, struct.pack(f"{len(words)}q", *words), n,
                                         N.raw_stream(device.index)), "gdn2_adamw_step")
    del lists["grads"]
    # autograd does not see the kernel's writes: a graph that saved one of these
    # tensors has to fail instead of differentiating with the new values
    increment_version(chain.from_iterable(lists.values()))


class AdamW(torch.optim.Optimizer):
    r"""AdamW with decoupled weight decay on :func:`adamw_step`.

    ``state_bits``: 32 (float32 moments) or 8 (e4m3 codes with a scale for each
    256 elements, a quarter of the memory).  ``master_weights`` keeps float32
    copies of 16-bit parameters, on which the steps are taken.  Parameters must
    be contiguous CUDA tensors; those without a gradient are skipped.
    """

    def __init__(self, params, lr: float = 1e-3, betas: tuple[float, float] = (0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float = 1e-2, *, state_bits: int = 32,
                 master_weights: bool = False):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32; got {state_bits}")
        if not (lr >= 0 and math.isfinite(lr)):
            raise ValueError(f"lr must be finite and not negative; got {lr}")
        if not all(0 <= b < 1 for b in betas):
            raise ValueError(f"betas must be in [0, 1); got {betas}")
        if not eps >= 0 or not weight_decay >= 0:
            raise ValueError("eps and weight_decay must not be negative")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay,
                                      state_bits=state_bits, master_weights=master_weights))

    def _state_of(self, p, group):
        s = self.state[p]
        if s:
            return s
        s["step"] = 0
        if group["state_bits"] == 8:
            blocks = -(-p.numel() // STATE_BLOCK)
            for k in ("exp_avg", "exp_avg_sq"):
                s[k] = torch.zeros(p.shape, dtype=torch.uint8, device=p.device).view(
                    torch.float8_e4m3fn)
                s[k + "_scale"] = torch.zeros(blocks, dtype=torch.float32, device=p.device)
        else:
            for k in ("exp_avg", "exp_avg_sq"):
                s[k] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
        if group["master_weights"] and p.dtype != torch.float32:
            s["master"] = p.detach().to(torch.float32, copy=True)
        return s

    @torch.no_grad()
    def step(self, closure=None, *, grad_scale: torch.Tensor | None = None,
             found_inf: torch.Tensor | None = None):
        """One step; ``grad_scale`` and ``found_inf`` as in :func:`adamw_step`
        (a step that ``found_inf`` leaves out is counted all the same)."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            batches: dict = {}  # what is counted and not yet taken
            try:
                for p in group["params"]:
                    if p.grad is None:
                        continue
                    if p.grad.is_sparse:
                        raise RuntimeError("AdamW (B200 build) does not take sparse gradients")
                    s = self._state_of(p, group)
                    s["step"] += 1
                    key = (p.device, p.dtype, p.grad.dtype, s["step"], "master" in s,
                           "exp_avg_scale" in s)
                    batches.setdefault(key, []).append((p, s))
                for key, items in list(batches.items()):
                    _, _, _, step, master, eight = key
                    of = lambda k: [s[k] for _, s in items]
                    adamw_step([p for p, _ in items], [p.grad for p, _ in items], of("exp_avg"),
                               of("exp_avg_sq"), step=step, lr=group["lr"], betas=group["betas"],
                               eps=group["eps"], weight_decay=group["weight_decay"],
                               exp_avg_scales=of("exp_avg_scale") if eight else None,
                               exp_avg_sq_scales=of("exp_avg_sq_scale") if eight else None,
                               master_params=of("master") if master else None,
                               grad_scale=grad_scale, found_inf=found_inf)
                    del batches[key]
            except BaseException:
                for items in batches.values():
                    for _, s in items:
                        s["step"] -= 1
                raise
        return loss

    def load_state_dict(self, state_dict):
        """As the base class, which casts states to their parameter's dtype;
        the moments keep the types they were saved with."""
        super().load_state_dict(state_dict)
        saved = state_dict["state"]
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(ids, params):
            for k, x in saved.get(i, {}).items():
                if isinstance(x, torch.Tensor):
                    self.state[p][k] = x.detach().to(device=p.device, copy=True).contiguous()
                else:
                    self.state[p][k] = x
