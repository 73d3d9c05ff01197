"""Dropout by a counter-based generator: the mask is drawn again in the backward instead of stored. No counterpart in the reference."""
from __future__ import annotations

import torch

from . import _native

_STREAM = 1 << 62   # counters that nothing else which draws from torch's generator reaches


def dropout(x: torch.Tensor, p: float = 0.5, seed: int | torch.Tensor | None = None, offset: int = 0, residual: torch.Tensor | None = None) -> torch.Tensor:
    """x with each element kept with probability 1 - p (met to 2^-17) and divided by it, zero otherwise, plus residual if there is one; in 32 bits, rounded
    once to x's type (float32, bfloat16 or float16), contiguous.

    Element i of x, in the order of its indices, has 16 bits of Philox4x32-10 (counter: i / 8 and `offset`, key: `seed`), so that the same numbers give the same mask
    whatever the type, and another offset (a layer's number, say) or seed another mask. seed: an int; or one int64 value on x's device, read
    when the kernels run and not to be changed before the backward (for a step captured into a graph: count it up within); or None, which
    draws seed and offset from the device's default torch generator (and advances it), outside a capture. A dropped element is 0 whatever x
    holds there. Differentiable with respect to x and residual; second and forward-mode derivatives raise."""
    if seed is None:
        if offset != 0:
            raise ValueError('efgs: an offset needs a seed')
        if x.device.type != 'cuda':
            raise ValueError(f"efgs: dropout's input must be on a GPU device, got {x.device}")
        with torch.cuda.device(x.device):
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError('efgs: a captured dropout needs its seed: the generator is read on the host')
        seed, drawn = _native.draw_counters(torch.cuda.default_generators[x.device.index])
        offset = drawn | _STREAM
    if not 0 <= offset < 1 << 64:
        raise ValueError(f'efgs: the offset must lie in [0, 2^64), got {offset}')
    if isinstance(seed, torch.Tensor):
        return _native.dropout(x, float(p), 0, seed, offset, residual)
    return _native.dropout(x, float(p), int(seed) & (1 << 64) - 1, None, offset, residual)
