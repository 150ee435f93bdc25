"""Float64 restatement of the AdamW step and of its 8-bit states (test
infrastructure): formulas written out, the format by its table of values."""

from __future__ import annotations

import numpy as np

BLOCK = 256
TOP_M, TOP_V = 448.0, 1.875


def table(bias, codes):
    """Values of the codes 0 .. codes - 1 of a format of 3 mantissa bits whose exponent
    field e stands for 2^(e - bias)."""
    c = np.arange(codes)
    e, f = c >> 3, c & 7
    return np.where(e > 0, (1 + f / 8) * 2.0 ** (e - bias), f / 8 * 2.0 ** (1 - bias))


TABLE_M, TABLE_V = table(7, 127), table(31, 256)


def decode(codes, scale, signed):
    codes = np.asarray(codes, np.int64).reshape(-1, BLOCK)
    if signed:
        x = np.where(codes & 128, -1.0, 1.0) * TABLE_M[codes & 127]
    else:
        x = TABLE_V[codes]
    return (x * np.asarray(scale, np.float64)[:, None]).ravel()


def words(seed, step, count):
    """A 32-bit word for each value: word i % 4 of the block with counter (i / 4, step)."""
    low = np.uint64(0xFFFFFFFF)
    half = np.uint64(32)
    block = np.arange((count + 3) // 4, dtype=np.uint64)
    c = [block & low, block >> half, np.full_like(block, step & 0xFFFFFFFF),
         np.full_like(block, step >> 32)]
    k = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> half) ^ c[1] ^ np.uint64(k[0]), p1 & low,
             (p0 >> half) ^ c[3] ^ np.uint64(k[1]), p0 & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, axis=1).astype(np.int64).ravel()[:count]


def encode(x, draws, signed):
    """(codes, scales) of values in blocks.  A block's scale is its largest value over the
    format's, rounded once; a value over the scale goes to the neighbour above with the
    probability of its way there."""
    x = np.asarray(x, np.float64).reshape(-1, BLOCK)
    values, top = (TABLE_M, TOP_M) if signed else (TABLE_V, TOP_V)
    most = np.abs(x).max(axis=1)
    scale = np.where(most >= 2.0 ** -120, most / top, 0.0).astype(np.float32)
    some = scale > 0
    a = np.where(some[:, None], np.abs(x) / np.where(some, scale, 1).astype(np.float64)[:, None], 0.0)
    below = np.clip(np.searchsorted(values, a, side="right") - 1, 0, len(values) - 1)
    above = np.minimum(below + 1, len(values) - 1)
    gap = np.where(above > below, values[above] - values[below], 1.0)
    up = (a - values[below]) / gap + (draws.reshape(x.shape) + 0.5) / 65536 >= 1
    code = np.where(up, above, below)
    if signed:
        code = code | np.where(x < 0, 128, 0)
    else:
        code = np.where((x > 0) & some[:, None], np.maximum(code, 1), code)
    return code.ravel(), scale


def moments(m, v, g, betas):
    return betas[0] * m + (1 - betas[0]) * g, betas[1] * v + (1 - betas[1]) * g * g


def update(p, m, v, rate, step, betas, eps, decay):
    c1, c2 = 1 - betas[0] ** step, 1 - betas[1] ** step
    return p * (1 - rate * decay) - rate * (m / c1) / (np.sqrt(v / c2) + eps)


def clip(grads, max_norm):
    """(norm, factor) of a list of gradients."""
    norm = np.sqrt(sum(float((np.asarray(g, np.float64) ** 2).sum()) for g in grads))
    return norm, (max_norm / norm if norm > max_norm else 1.0)
