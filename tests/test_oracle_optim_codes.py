"""The codes of the 8-bit states against rational arithmetic: the scale is the float32
nearest to the largest value over the format's, a code is decided by the quotient of a
value and that scale."""

from fractions import Fraction

import numpy as np
import pytest

from oracle import optim as oo
from oracle.layers import philox


def _code(value, scale, draw, table):
    """By the quotient as a fraction."""
    q = Fraction(float(abs(value))) / Fraction(float(scale))
    below = max(i for i, t in enumerate(table) if Fraction(float(t)) <= q)
    if below + 1 == len(table):
        return below
    low, high = Fraction(float(table[below])), Fraction(float(table[below + 1]))
    up = (q - low) / (high - low) + Fraction(2 * int(draw) + 1, 131072) >= 1
    return below + 1 if up else below


def near_borders(rng, blocks, table, top):
    """(values, draws): 255 values of each block lie a part in 10^9 on either side of where
    their draw begins to round them up, of scales of any size."""
    most = rng.uniform(1, 2, blocks) * 2.0 ** rng.integers(-40, 20, blocks)
    scale = (most / top).astype(np.float32).astype(np.float64)
    draws = rng.integers(0, 65536, (blocks, oo.BLOCK))
    code = rng.integers(len(table) // 2, len(table) - 2, (blocks, oo.BLOCK))
    border = table[code] + (table[code + 1] - table[code]) * (1 - (draws + 0.5) / 65536)
    x = border * scale[:, None] * (1 + 1e-9 * rng.choice([-1.0, 1.0], code.shape))
    x[:, 77] = most
    return x, draws


@pytest.mark.parametrize("signed", [True, False])
def test_scales_and_codes_are_those_of_the_quotients(signed, rng):
    table, top = (oo.TABLE_M, oo.TOP_M) if signed else (oo.TABLE_V, oo.TOP_V)
    x, draws = near_borders(rng, 12, table, top)
    code, scale = oo.encode(x, draws, signed)
    code = code.reshape(x.shape)
    for b in range(len(x)):
        exact = Fraction(float(np.abs(x[b]).max())) / Fraction(top)
        ulp = Fraction(float(np.spacing(scale[b])))
        assert abs(Fraction(float(scale[b])) - exact) <= ulp / 2 * (1 + Fraction(1, 1 << 20))
        assert all(_code(v, scale[b], d, table) == c
                   for v, d, c in zip(x[b], draws[b], code[b]))


@pytest.mark.parametrize("largest", [2.0 ** -120, 1.5 * 2.0 ** -120, 2.0 ** -119])
def test_the_smallest_blocks(largest):
    x = np.zeros(256)
    x[:4] = largest, -largest, largest / 2, -largest / 3
    for draw in (0, 65535):
        code, scale = oo.encode(x, np.full(256, draw), True)
        got = oo.decode(code, scale, True)
        assert not got[4:].any()
        # a scale below fp32's normal range has steps of 2^-149
        assert np.abs(got - x).max() <= largest / 8 + 448 * 2.0 ** -149
    code, scale = oo.encode(0.99 * x, np.full(256, 65535), True)
    assert (scale[0] == 0) == (0.99 * largest < 2.0 ** -120)


def test_words_are_the_generators():
    for seed, step in ((0, 1), ((1 << 63) + 5, 1000), ((1 << 64) - 1, (1 << 53) - 1)):
        want = [w for b in range(5) for w in philox(b | (step << 64), seed)]
        assert np.array_equal(oo.words(seed, step, 18), want[:18])
