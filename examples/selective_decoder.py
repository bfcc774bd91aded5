"""A small decoder of GDN-2 and selective state space layers, trained and sampled.

    python examples/selective_decoder.py [--steps 40]

* A selective layer is ``short_conv`` and ``selective_scan`` between projections; its
  prompt and its single tokens go through the same operators (``short_conv`` with the
  tokens before it, ``selective_scan_step`` on a state pool).
* The training step is ``token_logprobs``, ``grad_norm`` and ``AdamW``: the clipping
  coefficient, and whether the step is left out because a gradient is not finite,
  stay on the device.
* Serving runs the prompt at once, then samples one token at a time with
  ``sample_tokens``, every row by its own temperature, top-k and top-p.
"""

from __future__ import annotations

import argparse
import os
import sys

import torch
from torch import nn

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from qwendopamine_b200 import (  # noqa: E402
    AdamW, GatedDeltaNet2, grad_norm, sample_tokens, selective_scan, selective_scan_step,
    token_logprobs)
from qwendopamine_b200.gdn2_ops import short_conv  # noqa: E402

VOCAB, HIDDEN = 101, 128


class SelectiveLayer(nn.Module):
    """Projections, short convolution and selective scan with its gate."""

    def __init__(self, hidden: int, states: int = 16, width: int = 4, rank: int = 8):
        super().__init__()
        self.inner, self.states, self.rank = 2 * hidden, states, rank
        self.in_proj = nn.Linear(hidden, 2 * self.inner, bias=False)
        self.conv = nn.Conv1d(self.inner, self.inner, width, groups=self.inner)
        self.x_proj = nn.Linear(self.inner, rank + 2 * states, bias=False)
        self.dt_proj = nn.Linear(rank, self.inner, bias=False)
        self.dt_bias = nn.Parameter(torch.linspace(-4.0, -1.0, self.inner))
        self.A_log = nn.Parameter(torch.arange(1.0, states + 1).log().repeat(self.inner, 1))
        self.D = nn.Parameter(torch.ones(self.inner))
        self.out_proj = nn.Linear(self.inner, hidden, bias=False)

    def parts(self, h, before=None, want=False):
        """Operands of the scan for tokens ``h`` [B, T, hidden], and the convolution's
        last tokens."""
        x, z = self.in_proj(h).chunk(2, dim=-1)
        x, last = short_conv(x, self.conv.weight, self.conv.bias, prefix=before, output_final_state=want)
        dt, B, C = self.x_proj(x).split([self.rank, self.states, self.states], dim=-1)
        A = -self.A_log.float().exp()
        return (x, self.dt_proj(dt), A, B, C, self.D, z), last

    def forward(self, h):
        ops, _ = self.parts(h)
        y, _ = selective_scan(*ops, dt_bias=self.dt_bias, dt_softplus=True)
        return self.out_proj(y)

    def prompt(self, h, cache):
        """The same; ``cache`` (conv [S, W-1, D], pool [S, D, N]) holds the states behind it."""
        conv, pool = cache
        ops, last = self.parts(h, want=True)
        y, state = selective_scan(*ops, dt_bias=self.dt_bias, dt_softplus=True, output_final_state=True)
        conv.copy_(last.transpose(1, 2))
        pool.copy_(state)
        return self.out_proj(y)

    def step(self, h, cache, slots):
        """One token of each sequence: ``h`` [B, hidden]."""
        conv, pool = cache
        ops, last = self.parts(h[:, None], before=conv, want=True)
        conv.copy_(last.transpose(1, 2))
        one = [t[:, 0] if t.ndim == 3 else t for t in ops]
        return self.out_proj(selective_scan_step(*one, dt_bias=self.dt_bias, dt_softplus=True, state=pool,
                                                 state_indices=slots))

    def cache(self, rows):
        like = dict(device=self.D.device)
        return (torch.zeros(rows, self.conv.weight.shape[-1] - 1, self.inner, dtype=self.D.dtype, **like),
                torch.zeros(rows, self.inner, self.states, **like))


class Decoder(nn.Module):
    def __init__(self, layers: int = 3):
        super().__init__()
        self.embed = nn.Embedding(VOCAB, HIDDEN)
        self.norms = nn.ModuleList(nn.RMSNorm(HIDDEN) for _ in range(layers + 1))
        self.mixers = nn.ModuleList(
            GatedDeltaNet2(hidden_size=HIDDEN, num_heads=2, head_dim=64, layer_idx=i) if i % 2 else
            SelectiveLayer(HIDDEN) for i in range(layers))
        self.head = nn.Linear(HIDDEN, VOCAB, bias=False)

    def forward(self, ids):
        x = self.embed(ids)
        for norm, mix in zip(self.norms, self.mixers):
            y = mix(norm(x))
            x = x + (y if isinstance(mix, SelectiveLayer) else y[0])
        return self.head(self.norms[-1](x))

    def prompt(self, ids, caches):
        x = self.embed(ids)
        for norm, mix, cache in zip(self.norms, self.mixers, caches):
            if isinstance(mix, SelectiveLayer):
                x = x + mix.prompt(norm(x), cache)
            else:
                x = x + mix(norm(x), past_key_values=cache, use_cache=True)[0]
        return self.head(self.norms[-1](x[:, -1]))

    def step(self, ids, caches, slots):
        x = self.embed(ids)
        for norm, mix, cache in zip(self.norms, self.mixers, caches):
            h = norm(x)
            if isinstance(mix, SelectiveLayer):
                x = x + mix.step(h, cache, slots)
            else:
                x = x + mix(h[:, None], past_key_values=cache, use_cache=True)[0][:, 0]
        return self.head(self.norms[-1](x))

    def caches(self, rows):
        return [m.cache(rows) if isinstance(m, SelectiveLayer) else dict() for m in self.mixers]


def train_step(model, opt, ids, max_norm: float = 1.0):
    """One step on ``ids`` [rows, T + 1]; returns the loss and the gradients' norm,
    both on the device."""
    opt.zero_grad()
    loss = -token_logprobs(model(ids[:, :-1]), ids[:, 1:]).logprobs.mean()
    loss.backward()
    r = grad_norm([p.grad for p in model.parameters()], max_norm=max_norm)
    opt.step(grad_scale=r.clip_coef, found_inf=r.found_inf)
    return loss.detach(), r


@torch.no_grad()
def serve(model, prompt, new, uniform, **options):
    """``new`` sampled tokens behind each row of ``prompt`` [rows, T]; ``uniform``
    [new, rows], the options one value for each row."""
    rows = prompt.shape[0]
    caches, slots = model.caches(rows), torch.arange(rows, dtype=torch.int32, device=prompt.device)
    logits, ids = model.prompt(prompt, caches), []
    for t in range(new):
        ids.append(sample_tokens(logits, uniform[t], **options))
        if t + 1 < new:
            logits = model.step(ids[-1], caches, slots)
    return torch.stack(ids, 1)


def main(steps: int = 40) -> dict:
    device = torch.device("cuda")
    torch.manual_seed(0)
    model = Decoder().to(device, torch.bfloat16)
    opt = AdamW(model.parameters(), lr=2e-3, weight_decay=0.01, master_weights=True)
    gen = torch.Generator(device=device).manual_seed(0)
    losses, norms = [], []
    for _ in range(steps):
        start = torch.randint(0, VOCAB, (16, 1), generator=gen, device=device)
        ids = (start + 3 * torch.arange(65, device=device)) % VOCAB
        loss, r = train_step(model, opt, ids)
        losses.append(loss)
        norms.append(r.norm)
    model.eval()
    rows = 4
    options = dict(temperature=torch.tensor([0.0, 0.7, 1.0, 1.3], device=device),
                   top_k=torch.tensor([0, 20, 0, 50], dtype=torch.int32, device=device),
                   top_p=torch.tensor([1.0, 1.0, 0.9, 0.95], device=device))
    uniform = torch.rand(12, rows, generator=gen, device=device)
    prompt = (torch.arange(rows, device=device)[:, None] + 3 * torch.arange(20, device=device)) % VOCAB
    return dict(losses=torch.stack(losses).float().tolist(), norms=torch.stack(norms).tolist(),
                sampled=serve(model, prompt, 12, uniform, **options).tolist())


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=40)
    r = main(ap.parse_args().steps)
    print(f"loss {r['losses'][0]:.3f} -> {r['losses'][-1]:.3f}, gradient norm {r['norms'][-1]:.3f}")
    for row in r["sampled"]:
        print(*row)
