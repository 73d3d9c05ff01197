"""Losses that shared codes and tokens are learned with: the cross entropy of rows against a table, whose logits are never in memory, and the
balance of how often codes or experts are chosen. No counterpart in the reference."""
from __future__ import annotations

import torch

from . import _native


def linear_cross_entropy(features: torch.Tensor, table: torch.Tensor, targets: torch.Tensor, scale: float = 1.0, reduction: str = 'mean') -> torch.Tensor:
    """Softmax cross entropy of every feature row against all rows of a table: -log softmax(scale * features @ table.T)[target], float32.

    features: (..., columns); table: (rows, columns), both float32, bfloat16 or float16; targets: int32 or int64 of the features' shape
    without columns. A target outside [0, rows) (say -1 or -100) leaves its row out: its loss and gradient are zero, whatever its features hold.
    reduction: 'none' (a loss for each target), 'sum', or 'mean' over the rows that count (0 if none does). Logits, sums and statistics are in 32
    bits. Differentiable with respect to features and table, by pieces of the table whose logits are computed again; above 64 columns the logits'
    gradients are held in the inputs' type between the two products, but for what a row's own target's loses as it is rounded, which is added;
    of float16 with a loss for each target, to 2^-39 of the largest upstream gradient, so in fewer bits where a row's own is far smaller. Every sum
    has a fixed order, the same bits from call to call; second and forward-mode derivatives raise.

    Rows that count and the table should be finite: an infinity or NaN reaches the losses and gradients that its row has a part in, as NaN where
    float32 arithmetic might have left an infinity."""
    return _native.linear_cross_entropy(features, table, targets, float(scale), reduction)


def balance_loss(logits: torch.Tensor, indices: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(loss, counts) of choosing experts (or codes): E * sum over the E experts of (share of the choices) * (mean softmax probability), float32, 1 where
    both are even; counts: int64 (E,), how often each was chosen.

    logits: (..., E), E up to 8192, float32, bfloat16 or float16; indices: the chosen experts, int32 or int64, (...) or (..., choices), up to 65536. An index outside [0, E) counts
    nowhere, and a row without any other is left out (0 and zero gradients if all are). Differentiable with respect to the logits; the counts
    are not. Rows of nothing but -inf have no probabilities. Sums over rows are in a fixed order; second and forward-mode derivatives raise."""
    return _native.balance_loss(logits, indices)
