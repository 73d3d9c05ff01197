"""Learning which code follows which: the numbers of shared appearance codes along the primitives of a scene, as a sequence, say of primitives in the order of
a space-filling curve. A row of the codebook stands for the code before (`efgs.embedding`), dropout is drawn from a counter (`efgs.dropout`), a few experts, two
of them for each row, change it beside a residual (their choices balanced by `efgs.balance_loss`), and the next code is told from the same codebook
(`efgs.linear_cross_entropy`, no logits in memory). Codebook, router and experts are trained by `efgs.AdamW`.

The sequences are synthetic: a code mostly leads to one of four others; sequences end early, which padding of -1 marks.

    python examples/train_code_sequence.py --codes 4096 --sequences 64 --length 512 --steps 100
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'efficient-gaussian-appearance_amd'))

import efgs  # noqa: E402


def sequences(codes: int, count: int, length: int, seed: int) -> torch.Tensor:
    """(count, length) code numbers, -1 behind a sequence's end."""
    rng = torch.Generator().manual_seed(seed)
    follows = torch.randint(0, codes, (codes, 4), generator=rng)
    out = torch.empty(count, length, dtype=torch.int64)
    out[:, 0] = torch.randint(0, codes, (count,), generator=rng)
    for t in range(1, length):
        out[:, t] = follows[out[:, t - 1], torch.randint(0, 4, (count,), generator=rng)]
    end = torch.randint(length // 2, length + 1, (count, 1), generator=rng)
    return torch.where(torch.arange(length) < end, out, -1)


def parameters(codes: int, width: int, experts: int, seed: int, dtype: torch.dtype, device: torch.device) -> dict[str, torch.Tensor]:
    rng = torch.Generator().manual_seed(seed)
    shapes = dict(codebook=((codes, width), 1.0), router=((width, experts), width ** -0.5), experts=((width, experts * width), width ** -0.5))  # (side by side: one product)
    return {k: (torch.randn(shape, generator=rng) * scale).to(dtype).to(device) for k, (shape, scale) in shapes.items()}


def step_loss(p: dict[str, torch.Tensor], numbers: torch.Tensor, drop: float, seed: int, balance: float = 0.01) -> tuple[torch.Tensor, torch.Tensor]:
    """(loss, how often each expert was chosen) of predicting numbers[:, 1:] from numbers[:, :-1]."""
    before, after = numbers[:, :-1].reshape(-1), numbers[:, 1:].reshape(-1)
    width, experts = p['codebook'].shape[1], p['router'].shape[1]
    h = efgs.dropout(efgs.embedding(before, p['codebook']), drop, seed=seed, offset=0)
    logits = h @ p['router']
    chosen = logits.detach().float().topk(min(2, experts), dim=1).indices
    even, counts = efgs.balance_loss(logits, torch.where(before[:, None] >= 0, chosen, -1))
    gates = torch.zeros_like(logits).scatter(1, chosen, torch.softmax(logits.gather(1, chosen), 1))
    mixed = ((h @ p['experts']).view(-1, experts, width) * gates[:, :, None]).sum(1)
    out = efgs.dropout(mixed, drop, seed=seed, offset=1, residual=h)
    return efgs.linear_cross_entropy(out, p['codebook'], after, scale=width ** -0.5) + balance * even, counts


def train(codes: int = 4096, count: int = 64, length: int = 512, width: int = 64, experts: int = 8, steps: int = 100, drop: float = 0.1,
          dtype: torch.dtype = torch.float32, device: str = 'cuda:0', report: int = 0) -> list[float]:
    """The loss of every step."""
    dev = torch.device(device)
    numbers = sequences(codes, count, length, 0).to(dev)
    p = {k: t.requires_grad_() for k, t in parameters(codes, width, experts, 1, dtype, dev).items()}
    optimizer = efgs.AdamW(list(p.values()), lr=3e-3, weight_decay=1e-4, max_grad_norm=1.0)
    losses = []
    for step in range(steps):
        loss, counts = step_loss(p, numbers, drop, step)
        optimizer.zero_grad(set_to_none=True)
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
        if report and (step + 1) % report == 0:
            print(f'step {step + 1}: loss {float(losses[-1]):.4f}, choices of the experts {counts.tolist()}', flush=True)
    return [float(x) for x in losses]


if __name__ == '__main__':
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument('--codes', type=int, default=4096)
    ap.add_argument('--sequences', type=int, default=64)
    ap.add_argument('--length', type=int, default=512)
    ap.add_argument('--width', type=int, default=64)
    ap.add_argument('--experts', type=int, default=8)
    ap.add_argument('--steps', type=int, default=100)
    ap.add_argument('--type', choices=('float32', 'bfloat16', 'float16'), default='float32')
    a = ap.parse_args()
    train(a.codes, a.sequences, a.length, a.width, a.experts, a.steps, dtype=getattr(torch, a.type), report=max(1, a.steps // 10))
