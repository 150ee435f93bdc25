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

ROWS, WIDTH, HIDDEN = 1500, 250, 1100  # the tiled products, ragged in each size


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


@pytest.mark.parametrize("rows, hidden", [(3, 20), (1500, 1100)])  # by either kernel
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
def test_gelu_far_from_zero(kind, rows, hidden):
    """Up to the largest values it is g or 0, and its derivative 1 or 0."""
    far = np.array([30.0, 39.0, 41.0, 1e10, 1.8e19, 1.9e19, 1e25, 3e38])
    gate = np.resize(np.concatenate([far, -far, [np.inf]]), hidden)
    bg = torch.from_numpy(gate).to("cuda", kind)
    x, w = torch.zeros(rows, 8, device="cuda", dtype=kind), \
        torch.zeros(hidden, 8, device="cuda", dtype=kind)
    ones = torch.ones(hidden, device="cuda", dtype=kind)
    h = features.gated_layer(x, w, w, bg, ones, activation="gelu")
    want = torch.where(bg > 0, bg, torch.zeros_like(bg))
    assert torch.equal(h, want.expand(rows, hidden))
    g = features.gated_layer_backward(ones.expand(rows, hidden).contiguous(), x, w, w, bg, ones,
                                      activation="gelu")
    finite = torch.isfinite(bg)
    slopes = rows * (bg > 0).double()
    # bfloat16 rounds the sum over the rows
    assert torch.equal(g.db_gate[finite], slopes.to(kind)[finite])


# ---------------------------------------------------------------- float16

U16 = 2.0 ** -11


def _half(a):
    return torch.from_numpy(np.asarray(a)).to("cuda", torch.float16)


def _half_layer(rng, rows, width=64, hidden=128):
    return [_half(a) for a in (rng.normal(size=(rows, width)),
                               rng.normal(size=(hidden, width)) / np.sqrt(width),
                               rng.normal(size=(hidden, width)) / np.sqrt(width),
                               0.3 * rng.normal(size=hidden), 0.3 * rng.normal(size=hidden))]


def _half_check(got, want, tol, axis=None):
    """On the 2-norm of the whole result or of each row, entries that pass 65504
    (infinite in float16) among it: the roundings of dg and du that meet in an entry
    are those of terms as large as in any other.  A result's own rounding is absolute
    below 2^-14."""
    got = got.double().cpu().numpy()
    inside = abs(want) < 65504 * (1 - 2 * tol)
    assert np.all(np.isfinite(got[inside])) and np.all(abs(got[abs(want) > 65536]) > 65000)
    count = want.size if axis is None else want.shape[axis]
    err = np.linalg.norm(np.where(inside, got, 0.0) - np.where(inside, want, 0.0), axis=axis)
    assert np.all(err <= tol * np.linalg.norm(want, axis=axis) + 2.0 ** -25 * np.sqrt(count))


@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid", "relu"])
@pytest.mark.parametrize("rows", [100, 3000])
@pytest.mark.parametrize("size", [1e4, 1.0, 1e-5, 4e-6])
def test_float16_gradients_of_any_size(size, rows, act):
    """dg and du pass float16's largest and smallest values long before the
    gradients formed from them do.  Units of rounding as in test_gpu_torch_layers."""
    rng = np.random.default_rng(rows)
    args = _half_layer(rng, rows)
    dh = _half(size * rng.normal(size=(rows, 128)))
    got = features.gated_layer_backward(dh, *args, activation=act)
    host = [a.double().cpu().numpy() for a in (dh, *args)]
    for g, want, units in zip(got, ol.gated_layer_backward(*host, act=act), (3, 2, 2, 1, 1)):
        _half_check(g, want, units * U16 + 4e-6)


@pytest.mark.parametrize("rows", [100, 3000])
def test_float16_rows_of_different_sizes(rows):
    """dx, row by row, with rows of dh and of x 2^27 and 2^16 apart, some of dh zero."""
    rng = np.random.default_rng(5)
    args = _half_layer(rng, rows)
    args[0] *= _half(2.0 ** rng.integers(-8, 9, size=(rows, 1)))
    dh = 2.0 ** rng.integers(-14, 14, size=(rows, 1)) * rng.normal(size=(rows, 128))
    dh[::17] = 0.0
    dh = _half(dh)
    args[0][17, 3] = float("inf")  # of a row that has no gradient
    got = features.gated_layer_backward(dh, *args, need_dw=False)
    host = [a.double().cpu().numpy() for a in (dh, *args)]
    host[1][17, 3] = 0.0
    want = ol.gated_layer_backward(*host)[0]
    keep = np.arange(rows) != 17
    _half_check(got.dx[torch.from_numpy(keep).cuda()], want[keep], 3 * U16 + 4e-6, axis=1)


def test_float16_without_gradient():
    rng = np.random.default_rng(6)
    args = _half_layer(rng, 300)
    for g in features.gated_layer_backward(torch.zeros(300, 128, device="cuda").half(), *args):
        assert not g.any()
