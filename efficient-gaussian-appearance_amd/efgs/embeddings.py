"""Rows of a table by index, scaled: shared appearance codes of primitives, or any other embedding. No counterpart in the
reference, whose features are one row per primitive."""
from __future__ import annotations

import torch

from . import _native


def embedding(indices: torch.Tensor, table: torch.Tensor, scale: float = 1.0, padding_idx: int | None = None) -> torch.Tensor:
    """scale * table[indices]: (*indices.shape, columns) in the table's type, scaled in 32 bits and rounded once.

    indices: int32 or int64 of any shape; one outside [0, rows) (say -1: a primitive without a code) gives a zero row and gets no
    gradient. table: (rows, columns) float32, bfloat16 or float16. Differentiable with respect to the table: a row's gradient is
    scale times the sum of the upstream rows that it went to, added in 32 bits in a fixed order that the indices and sizes give, the same bit for bit
    from call to call; second and forward-mode derivatives raise. The row `padding_idx` is looked up like any other and gets no gradient."""
    return _native.embedding(indices, table, float(scale), padding_idx)
