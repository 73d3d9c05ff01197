"""The training operators in 64 bits from their definitions, for the tests: AdamW with 32-bit and 8-bit states, the coding of
8-bit states, the lookup of table rows and its gradient. Plain numpy on the CPU, without the library's code."""
from __future__ import annotations

import numpy as np

ROOT = dict(c=2.0 ** -16, exponent=-16, codes=256)   # r = sqrt(v) against its block's scale
RATIO = dict(c=2.0 ** -8, exponent=-8, codes=128)    # |m| / sqrt(v) against its bound
TOP = 31 / 32                                        # the top codes' y + c


def ratio_bound(beta1: float, beta2: float) -> float:
    return (1 - beta1) / np.sqrt((1 - beta2) * (1 - beta1 ** 2 / beta2))


def code_value(code, kind):
    """Value of a code: y + c has 16 codes to an octave, the first at c."""
    code = np.asarray(code, np.int64)
    return (1 + (code % 16) / 16) * 2.0 ** (code // 16 + kind['exponent']) - kind['c']


def code_position(y, kind):
    """Real-valued code of y >= 0: whole numbers at code_value's values, linear between them."""
    z = np.asarray(y, np.float64) + kind['c']
    exponent = np.floor(np.log2(z)).astype(np.int64)
    exponent -= z < 2.0 ** exponent
    exponent += z >= 2.0 ** (exponent + 1)
    return (exponent - kind['exponent'] + z / 2.0 ** exponent - 1) * 16


def mix(x):
    x = np.asarray(x, np.uint64) & np.uint64(0xffffffff)
    for shift, factor in ((16, 0x6C8E9CF5), (15, 0x3A2F4D1B)):
        x = ((x ^ (x >> np.uint64(shift))) * np.uint64(factor)) & np.uint64(0xffffffff)
    return x ^ (x >> np.uint64(16))


def dither(n: int, step: int, seed: int, first: int = 0):
    """Dithers of root and ratio of elements first..first + n, in [0, 1)."""
    key = mix(mix(seed) + np.uint64(step))
    i = np.arange(first, first + n, dtype=np.uint64) & np.uint64(0xffffffff)
    h = mix(((i * np.uint64(0x9E3779B1)) & np.uint64(0xffffffff)) + key)
    return (h & np.uint64(0xffff)).astype(np.float64) / 65536, (h >> np.uint64(16)).astype(np.float64) / 65536


def decode(ratio, root, scale, bound: float):
    """(m, v, u, r) of 8-bit states."""
    r = code_value(root, ROOT) * np.repeat(np.asarray(scale, np.float64), 256)[:len(root)]
    u = code_value(np.asarray(ratio) & 127, RATIO) * bound / (TOP - RATIO['c']) * np.where(np.asarray(ratio) >= 128, -1.0, 1.0)
    return u * r, r * r, u, r


def encode_positions(m, v, bound: float):
    """(positions of |u|, positions of r, scales, u's sign) of what a step would code, before the dither."""
    r = np.sqrt(v)
    r = np.where(np.isfinite(r), r, 0.0)
    n = len(r)
    scale = np.pad(r, (0, -n % 256)).reshape(-1, 256).max(1) / (TOP - ROOT['c'])
    scale = np.where(scale < 2.0 ** -100, 0.0, scale)
    full = np.repeat(scale, 256)[:n]
    with np.errstate(all='ignore'):
        root = code_position(np.where(full > 0, r / full, 0.0), ROOT)
        u = np.where(r > 0, m / r, 0.0)
    ratio = code_position(np.minimum(np.abs(u) / bound * (TOP - RATIO['c']), TOP - RATIO['c']), RATIO)
    return ratio, root, scale, u < 0


def adamw(p, g, m, v, step: int, lrs, beta1: float, beta2: float, eps: float, weight_decay: float, coefficient: float = 1.0):
    """(p, m, v) after a step."""
    g = np.asarray(g, np.float64) * coefficient
    m = beta1 * m + (1 - beta1) * g
    v = beta2 * v + (1 - beta2) * g * g
    lr = np.resize(np.asarray(lrs, np.float64), len(p)) if np.ndim(lrs) else float(lrs)
    with np.errstate(all='ignore'):
        update = (m / (1 - beta1 ** step)) / (np.sqrt(v / (1 - beta2 ** step)) + eps)
    return np.asarray(p, np.float64) * (1 - lr * weight_decay) - lr * update, m, v


def clip_coefficient(grads, max_norm: float) -> tuple[float, float]:
    norm = float(np.sqrt(sum(float((np.asarray(g, np.float64) ** 2).sum()) for g in grads)))
    return norm, min(1.0, max_norm / (norm + 1e-6))


def embedding(indices, table, scale: float):
    indices, table = np.asarray(indices).reshape(-1), np.asarray(table, np.float64)
    out = np.zeros((len(indices), table.shape[1]))
    inside = (indices >= 0) & (indices < len(table))
    out[inside] = table[indices[inside]] * scale
    return out


def embedding_gradient(indices, grad_out, rows: int, scale: float, padding=None):
    """(gradient, sum of magnitudes per value, entries per row)."""
    indices, grad_out = np.asarray(indices).reshape(-1), np.asarray(grad_out, np.float64)
    inside = (indices >= 0) & (indices < rows)
    if padding is not None:
        inside &= indices != padding
    total, magnitude = np.zeros((rows, grad_out.shape[1])), np.zeros((rows, grad_out.shape[1]))
    np.add.at(total, indices[inside], grad_out[inside])
    np.add.at(magnitude, indices[inside], np.abs(grad_out[inside]))
    return total * scale, magnitude * abs(scale), np.bincount(indices[inside], minlength=rows)
