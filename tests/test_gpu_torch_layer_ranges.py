"""The gated layer on values of different sizes in one array, entry by entry.

Bounds.  A sum of n products in fp32 by matrix instructions of 32 products, six
instructions each where an operand goes in three parts, is off by at most
SUM(n) = 2^-23 (6 n / 32 + 10) of the sum of the products' sizes (one rounding an
instruction, doubled for those inside one, and a few for parts that are left
out).  What that makes of g and u goes on through the formulas to first order:
|act'| <= 1.13, |act''| <= 1, and 3e-6 for the activation's own error (fp32)."""

import numpy as np
import pytest
import torch

from mojogp_amd import features
from oracle import layers as ol

pytestmark = pytest.mark.gpu

ROWS, WIDTH, HIDDEN = 1500, 250, 600  # the tiled products, ragged in each size


def _sum_bound(n):
    return 2.0 ** -23 * (6 * n / 32 + 10)


def _sizes(rng, n, decades):
    return 10.0 ** rng.uniform(-decades, decades, n)


def _spread(case, rng):
    """(x, w_gate, w_up, dh) of the sizes that the case is about, in float64 on
    the float32 grid."""
    x = rng.normal(size=(ROWS, WIDTH))
    wg, wu = (rng.normal(size=(HIDDEN, WIDTH)) / np.sqrt(WIDTH) for _ in range(2))
    dh = rng.normal(size=(ROWS, HIDDEN))
    if case == "outlier":
        x[7] *= 1e12
    elif case == "rows":
        x *= _sizes(rng, ROWS, 8)[:, None]
    elif case == "columns":  # features in units of their own
        c = _sizes(rng, WIDTH, 8)
        x, wg, wu = x * c, wg / c, wu / c
    elif case == "weight rows":
        wg, wu = wg * _sizes(rng, HIDDEN, 4)[:, None], wu * _sizes(rng, HIDDEN, 4)[:, None]
    elif case == "dh rows":
        dh *= _sizes(rng, ROWS, 8)[:, None]
    elif case == "dh columns":
        dh *= _sizes(rng, HIDDEN, 8)
    return tuple(a.astype(np.float32).astype(np.float64) for a in (x, wg, wu, dh))


def _bounds(x, wg, wu, bg, bu, dh, act):
    """What h and each gradient may be off by, entry by entry."""
    ax, ag, au = abs(x), abs(wg), abs(wu)
    own, near = _sum_bound(WIDTH), 3e-6
    g, u = x @ wg.T + bg, x @ wu.T + bu
    eg, eu = own * (ax @ ag.T + abs(bg)), own * (ax @ au.T + abs(bu))
    a, slope = ol.activate(act, g)
    ea = 1.13 * eg + near * abs(a)
    es = np.minimum(eg, 1.2) + near
    h = ea * (abs(u) + eu) + abs(a) * eu + 2.0 ** -22 * abs(a * u)
    dg, du = abs(dh * u * slope), abs(dh * a)
    edg = abs(dh) * (es * (abs(u) + eu) + abs(slope) * eu) + 2.0 ** -22 * dg
    edu = abs(dh) * ea + 2.0 ** -22 * du
    back, over = _sum_bound(2 * HIDDEN), _sum_bound(ROWS)
    dx = (edg + back * dg) @ ag + (edu + back * du) @ au
    rows = 2.0 ** -24 * ROWS  # the bias gradients: fp32 additions
    return h, (dx, (edg + over * dg).T @ ax, (edu + over * du).T @ ax,
               (edg + rows * dg).sum(axis=0), (edu + rows * du).sum(axis=0))


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("case", ["outlier", "rows", "columns", "weight rows", "dh rows",
                                  "dh columns"])
def test_float32_of_different_sizes(case, act):
    """A row's result does not depend on how large the rows, columns and weights
    beside it are."""
    rng = np.random.default_rng(11)
    x, wg, wu, dh = _spread(case, rng)
    bg, bu = (rng.normal(size=HIDDEN).astype(np.float32).astype(np.float64) for _ in range(2))
    args = [torch.from_numpy(a).to("cuda", torch.float32) for a in (x, wg, wu, bg, bu)]
    h = features.gated_layer(*args, activation=act)
    grads = features.gated_layer_backward(torch.from_numpy(dh).to("cuda", torch.float32), *args,
                                          activation=act)
    eh, eg = _bounds(x, wg, wu, bg, bu, dh, act)
    want = ol.gated_layer(x, wg, wu, bg, bu, act=act)
    assert np.all(abs(h.double().cpu().numpy() - want) <= eh + 1e-35)
    for name, got, ref, bound in zip(grads._fields, grads,
                                     ol.gated_layer_backward(dh, x, wg, wu, bg, bu, act=act), eg):
        assert np.all(abs(got.double().cpu().numpy() - ref) <= bound + 1e-35), name


def test_float32_non_finite_rows_stay_their_own():
    """As the few-row kernel, the tiled products leave every other row as it is."""
    rng = np.random.default_rng(12)
    x, wg, wu, _ = _spread("plain", rng)
    args = [torch.from_numpy(a).to("cuda", torch.float32) for a in (x, wg, wu)]
    clean = features.gated_layer(*args)
    args[0][3, 5] = float("nan")
    args[0][1400, 249] = float("inf")
    args[0][700, 0] = 3.4e38  # rounds to infinity in 16 bits
    got = features.gated_layer(*args)
    keep = [r for r in range(ROWS) if r not in (3, 700, 1400)]
    assert torch.equal(got[keep], clean[keep])
    assert torch.isnan(got[3]).all() and not torch.isfinite(got[1400]).all()
    g, u = x[700] @ wg.T + (3.4e38 - x[700, 0]) * wg[:, 0], \
        x[700] @ wu.T + (3.4e38 - x[700, 0]) * wu[:, 0]
    with np.errstate(over="ignore"):
        want = np.where(g > 0, g * u, 0.0).astype(np.float32)  # silu of +-1e37
    assert np.array_equal(np.isinf(want), np.isinf(got[700].cpu().numpy()))
    assert np.array_equal(np.sign(want), np.sign(got[700].cpu().numpy()))
