"""The kernels that serve large layers and point sets, which the smaller tests do not
reach: the gated layer's tiled products with every activation, type, stride and bias,
their 256 x 256 tiles in each backward product, and the points' gradient with four row
tiles a wave.

The gated layer's reference is its formulas in float64 tensor operations on the device;
tolerances as in test_gpu_torch_layers and test_gpu_torch_input_gradient."""

import math

import numpy as np
import pytest
import torch

from mojogp_amd import features
from mojogp_amd._provider import NativeProvider

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
UNIT = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
F32 = 4e-6
TOL = 4e-6


def _layer(rows, width, hidden, kind, pad=0, seed=0):
    """(x, w_gate, w_up, b_gate, b_up, dh), rows of tables `pad` columns wider, with
    NaN beside them."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(rows + width + hidden + seed)

    def matrix(r, c, scale=1.0):
        wide = torch.full((r, c + pad), float("nan"), device="cuda", dtype=TYPES[kind])
        view = wide[:, min(pad, 1):min(pad, 1) + c]
        view.copy_(scale * torch.randn(r, c, device="cuda", generator=gen))
        return view

    bias = [(0.3 * torch.randn(hidden, device="cuda", generator=gen)).to(TYPES[kind])
            for _ in range(2)]
    return [matrix(rows, width), matrix(hidden, width, width ** -0.5),
            matrix(hidden, width, width ** -0.5), *bias, matrix(rows, hidden)]


def _formulas(x, wg, wu, bg, bu, dh, act):
    """(h, dx, dw_gate, dw_up, db_gate, db_up) in float64."""
    x, wg, wu, dh = (a.double().contiguous() for a in (x, wg, wu, dh))
    g = x @ wg.T + (0.0 if bg is None else bg.double())
    u = x @ wu.T + (0.0 if bu is None else bu.double())
    if act == "relu":
        a, slope = g.clamp(min=0.0), (g > 0).double()
    elif act == "gelu":
        cdf = 0.5 * torch.erfc(-g / math.sqrt(2.0))
        a, slope = g * cdf, cdf + g * torch.exp(-0.5 * g * g) / math.sqrt(2.0 * math.pi)
    else:
        s = torch.sigmoid(g)
        a, slope = (g * s, s * (1 + g * (1 - s))) if act == "silu" else (s, s * (1 - s))
    dg, du = dh * u * slope, dh * a
    return (a * u, dg @ wg + du @ wu, dg.T.contiguous() @ x, du.T.contiguous() @ x,
            dg.sum(dim=0), du.sum(dim=0))


def _check(got, want, units, kind):
    assert got.shape == want.shape and got.dtype == TYPES[kind]
    err = float((got.double() - want).norm())
    assert err <= (units * UNIT[kind] + F32) * float(want.norm())


def _check_layer(args, act, kind, biased=True):
    *layer, dh = args
    if not biased:
        layer[3:] = [None, None]
    want = _formulas(*layer, dh, act)
    _check(features.gated_layer(*layer, activation=act), want[0], 1, kind)
    grads = features.gated_layer_backward(dh, *layer, activation=act)
    for got, ref, units in zip(grads, want[1:], (3, 2, 2, 1, 1)):
        if got is not None:
            _check(got, ref, units, kind)


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("act", sorted(features.ACTIVATIONS))
@pytest.mark.parametrize("width, pad", [(72, 0), (250, 0), (200, 8), (131, 1)])
def test_tiled_products(kind, act, width, pad):
    """More workgroups than the few-row kernel takes; rows direct loads can and
    cannot take, with and without biases."""
    _check_layer(_layer(1501, width, 1103, kind, pad), act, kind, biased=pad != 8)


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("act", sorted(features.ACTIVATIONS))
def test_large_tiles_of_the_projections_and_dx(kind, act):
    _check_layer(_layer(16500, 500, 260, kind), act, kind)


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("rows, width, hidden, pad", [(8191, 1023, 2049, 1), (8200, 1030, 1000, 0),
                                                      (40003, 256, 1029, 0)])
def test_large_tiles_of_every_product(kind, rows, width, hidden, pad):
    """Weight gradients and dx by large tiles, whole and in parts, ragged."""
    act = ("gelu", "silu", "sigmoid")[rows % 3]
    _check_layer(_layer(rows, width, hidden, kind, pad), act, kind)


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("rows, width, hidden", [(1501, 250, 1103), (32760, 96, 1279)])
def test_tiled_products_keep_non_finite_rows_apart(kind, rows, width, hidden):
    x, *weights, dh = _layer(rows, width, hidden, kind)
    clean = features.gated_layer(x, *weights)
    before = features.gated_layer_backward(dh, x, *weights, need_dw=False).dx
    bad = [3, rows // 2, rows - 1]
    x[bad[0], 5], x[bad[1], 0], dh[bad[2], 7] = float("nan"), float("inf"), float("nan")
    got = features.gated_layer(x, *weights)
    after = features.gated_layer_backward(dh, x, *weights, need_dw=False).dx
    keep = torch.ones(rows, dtype=torch.bool, device="cuda")
    keep[bad] = False
    assert torch.equal(got[keep], clean[keep]) and torch.equal(after[keep], before[keep])
    assert torch.isnan(got[bad[0]]).all() and not torch.isfinite(got[bad[1]]).all()
    assert torch.isnan(after[[bad[0], bad[2]]]).all()


# ---------------------------------------------------------------- the points' gradient

def _points(n, d, t, seed=0):
    rng = np.random.default_rng([n, d, t, seed])
    X = rng.normal(size=(n, d)).astype(np.float32)
    params = np.append(1.5 * np.sqrt(d) * rng.uniform(0.6, 1.2, size=d), 1.3).astype(np.float32)
    return X, params, *(rng.normal(size=(t, n)).astype(np.float32) for _ in range(2))


def _sampled(kind, X, params, L, R, rows):
    """The float64 formula at some rows."""
    X, L, R = (a.astype(np.float64) for a in (X, L, R))
    ls = params[:-1].astype(np.float64)
    z = X / ls
    df = z[rows][:, None, :] - z[None]
    r2 = (df ** 2).sum(axis=2)
    u = np.sqrt(r2 * {"rbf": 1.0, "matern12": 1.0, "matern32": 3.0, "matern52": 5.0}[kind])
    e = np.exp(np.maximum(-u, -20.0))
    if kind == "rbf":
        h = np.exp(-0.5 * r2)
    elif kind == "matern12":
        h = np.divide(e, u, out=np.zeros_like(u), where=u > 0)
    else:
        h = 3.0 * e if kind == "matern32" else 5.0 / 3.0 * (1.0 + u) * e
    h *= L[:, rows].T @ R + R[:, rows].T @ L
    return -params[-1] / ls * (h[:, None, :] @ df)[:, 0]


def _gradient(kind, X, params, L, R):
    p = NativeProvider(kind, True, X, params, 0.1)
    try:
        return p.input_gradient(L, R)
    finally:
        p.close()


@pytest.mark.parametrize("kind", ["rbf", "matern32", "matern52"])
@pytest.mark.parametrize("n, d, t", [(25100, 8, 11), (25001, 1, 3), (26003, 5, 17), (20011, 2, 16),
                                     (12001, 12, 7), (9000, 24, 2)])
def test_matrix_cores_over_many_points(kind, n, d, t):
    """Row tiles two and four a wave; the route is the matrix cores': a point so far
    away that its norm sends the same set to the differences changes the bits."""
    X, params, L, R = _points(n, d, t)
    got = _gradient(kind, X, params, L, R)
    rows = np.arange(0, n, n // 150)
    want = _sampled(kind, X, params, L, R, rows)
    assert np.linalg.norm(got[rows] - want) <= TOL * np.linalg.norm(want)
    far = np.vstack([X, np.full((1, d), 400.0, np.float32)])
    none = np.zeros((t, 1), np.float32)
    other = _gradient(kind, far, params, np.hstack([L, none]), np.hstack([R, none]))[:-1]
    assert not np.array_equal(got, other)
    assert np.linalg.norm(other[rows] - want) <= TOL * np.linalg.norm(want)


@pytest.mark.parametrize("n, d, t", [(5003, 3, 11), (9001, 9, 16), (30001, 2, 3)])
def test_matern12_over_many_points(n, d, t):
    X, params, L, R = _points(n, d, t)
    got = _gradient("matern12", X, params, L, R)
    rows = np.arange(0, n, n // 150)
    want = _sampled("matern12", X, params, L, R, rows)
    assert np.linalg.norm(got[rows] - want) <= TOL * np.linalg.norm(want)
