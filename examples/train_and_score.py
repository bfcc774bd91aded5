"""A small decoder trained and served with the operators around the GDN-2 mixer.

    python examples/train_and_score.py [--steps 60]

The decoder alternates :class:`~qwendopamine_b200.GatedDeltaNet2` layers with
gated linear recurrences (``gated_scan``) and learns to step along a fixed walk
through its vocabulary, a token depending on the two before it:

* the loss is ``token_logprobs`` of the targets (prompt tokens ignored) with a
  small entropy bonus;
* the step is ``AdamW`` with 8-bit states and fp32 master weights, its gradients
  scaled by a clipping coefficient that stays on the device;
* serving feeds one token at a time through both kinds of layer (the mixer's
  cache, and ``gated_scan_step`` on a state pool) and reports each chosen
  token's log probability with its best alternatives.
"""

from __future__ import annotations

import argparse
import os
import sys

import torch
import torch.nn.functional as F
from torch import nn

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from qwendopamine_b200 import (  # noqa: E402
    AdamW, GatedDeltaNet2, gated_scan, gated_scan_step, grad_norm, token_logprobs)

VOCAB, HIDDEN, IGNORE = 97, 128, -100


class GatedRecurrence(nn.Module):
    """Projections around the gated linear recurrence: value, decay, write gate."""

    def __init__(self, hidden: int):
        super().__init__()
        self.proj = nn.Linear(hidden, 3 * hidden, bias=False)
        self.decay_bias = nn.Parameter(torch.linspace(1.0, 6.0, hidden))
        self.out = nn.Linear(hidden, hidden, bias=False)

    def gates(self, x):
        v, g, w = self.proj(x).chunk(3, dim=-1)  # slices: the operator reads strided rows
        return v, F.logsigmoid(g.float() + self.decay_bias.float()), torch.sigmoid(w)

    def forward(self, x):
        v, g, w = self.gates(x)
        y, _ = gated_scan(v, g, w)
        return self.out(y)

    def step(self, x, pool, slots):
        v, g, w = self.gates(x)
        return self.out(gated_scan_step(v, g, w, state=pool, state_indices=slots))


class Decoder(nn.Module):
    def __init__(self, layers: int = 4):
        super().__init__()
        self.embed = nn.Embedding(VOCAB, HIDDEN)
        self.norms = nn.ModuleList(nn.RMSNorm(HIDDEN) for _ in range(layers + 1))
        self.mixers = nn.ModuleList(
            GatedDeltaNet2(hidden_size=HIDDEN, num_heads=2, head_dim=64, layer_idx=i) if i % 2 == 0
            else GatedRecurrence(HIDDEN) for i in range(layers))
        self.head = nn.Linear(HIDDEN, VOCAB, bias=False)

    def forward(self, ids):
        x = self.embed(ids)
        for norm, mix in zip(self.norms, self.mixers):
            y = mix(norm(x))
            x = x + (y[0] if isinstance(y, tuple) else y)
        return self.head(self.norms[-1](x))

    def step(self, ids, caches, slots):
        """Logits of one new token for each sequence; ``caches`` move on."""
        x = self.embed(ids)
        for norm, mix, cache in zip(self.norms, self.mixers, caches):
            h = norm(x)
            if isinstance(mix, GatedDeltaNet2):
                y = mix(h[:, None], past_key_values=cache, use_cache=True)[0][:, 0]
            else:
                y = mix.step(h, cache, slots)
            x = x + y
        return self.head(self.norms[-1](x))


def walk(ids, length):
    """``ids`` ``[rows, 2]`` continued to ``length`` tokens."""
    cols = [ids[:, 0], ids[:, 1]]
    while len(cols) < length:
        cols.append((7 * cols[-1] + 3 * (cols[-2] % 2)) % VOCAB)
    return torch.stack(cols, 1)


def batch(gen, rows, length, device):
    """Inputs and targets of walks from random starts; the second token cannot be
    known and bears no loss."""
    ids = walk(torch.randint(0, VOCAB, (rows, 2), generator=gen), length + 1).to(device)
    targets = ids[:, 1:].clone()
    targets[:, 0] = IGNORE
    return ids[:, :-1], targets


def train(model, steps, device):
    opt = AdamW(model.parameters(), lr=3e-3, betas=(0.9, 0.95), weight_decay=0.01, state_bits=8,
                master_weights=True)
    gen = torch.Generator().manual_seed(0)
    first = last = None
    for _ in range(steps):
        ids, targets = batch(gen, 32, 96, device)
        opt.zero_grad()
        r = token_logprobs(model(ids), targets, entropy=True, ignore_index=IGNORE)
        kept = (targets != IGNORE).sum()
        loss = -(r.logprobs.sum() + 1e-3 * r.entropy.sum()) / kept
        loss.backward()
        r = grad_norm([p.grad for p in model.parameters()], max_norm=1.0)
        opt.step(grad_scale=r.clip_coef, found_inf=r.found_inf)  # clipped on the device
        last = loss.detach()
        first = last if first is None else first
    return float(first), float(last)


@torch.no_grad()
def serve(model, prompt, new, device):
    """Greedy continuation of each prompt; returns ids and what is reported for
    the new tokens."""
    rows = prompt.shape[0]
    slots = torch.arange(rows, dtype=torch.int32, device=device)
    caches = [dict() if isinstance(m, GatedDeltaNet2) else torch.zeros(rows, HIDDEN, device=device)
              for m in model.mixers]
    ids, report = prompt, []
    for t in range(prompt.shape[1] + new - 1):
        logits = model.step(ids[:, t], caches, slots)
        if t >= prompt.shape[1] - 1:
            chosen = logits.argmax(-1)
            report.append(token_logprobs(logits, chosen, top_k=3, entropy=True))
            ids = torch.cat([ids, chosen[:, None]], 1)
    return ids, report


def main(steps: int = 60) -> dict:
    device = torch.device("cuda")
    torch.manual_seed(0)
    model = Decoder().to(device, torch.bfloat16)
    first, last = train(model, steps, device)
    model.eval()
    gen = torch.Generator().manual_seed(1)
    ids, _ = batch(gen, 4, 24, device)
    out, report = serve(model, ids[:, :12], 12, device)
    right = float((out[:, 12:] == ids[:, 12:]).float().mean())
    chosen = torch.stack([r.logprobs for r in report])
    best = torch.stack([r.top_logprobs[..., 0] for r in report])
    return dict(first=first, last=last, right=right, chosen=float(chosen.mean()),
                greedy_is_best=bool(torch.equal(chosen, best)))


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=60)
    r = main(ap.parse_args().steps)
    print(f"loss {r['first']:.3f} -> {r['last']:.3f}; {100 * r['right']:.0f} % of the continuation "
          f"right, mean log probability {r['chosen']:.3f}")
