"""The float64 layers that the kernels are compared with, pinned on their own:
gradients against central differences, the counter generator against its
published answers."""

import numpy as np
import pytest

from oracle import layers as ol

STEP = 1e-5
# central differences in float64: truncation STEP^2 f''' ~ 1e-10, rounding
# 1e-16 / STEP ~ 1e-11 of the function's size, a few hundred terms
TOL = 2e-7


def _differences(f, a):
    out = np.zeros_like(a)
    for i in np.ndindex(a.shape):
        p, m = a.copy(), a.copy()
        p[i] += STEP
        m[i] -= STEP
        out[i] = (f(p) - f(m)) / (2 * STEP)
    return out


def _close(got, want):
    assert np.linalg.norm(got - want) <= TOL * (1.0 + np.linalg.norm(want))


def test_layer_norm_gradients(rng):
    x, w, b = rng.normal(size=(4, 7)), rng.normal(size=7), rng.normal(size=7)
    dy = rng.normal(size=(4, 7))
    dx, dw, db = ol.layer_norm_backward(dy, x, w)
    _close(dx, _differences(lambda a: (dy * ol.layer_norm(a, w, b)).sum(), x))
    _close(dw, _differences(lambda a: (dy * ol.layer_norm(x, a, b)).sum(), w))
    _close(db, _differences(lambda a: (dy * ol.layer_norm(x, w, a)).sum(), b))


@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid", "relu"])
def test_gated_layer_gradients(rng, act):
    args = [rng.normal(size=s) for s in ((5, 3), (4, 3), (4, 3), (4,), (4,))]
    dh = rng.normal(size=(5, 4))
    for k, got in enumerate(ol.gated_layer_backward(dh, *args, act=act)):
        def f(a, k=k):
            return (dh * ol.gated_layer(*args[:k], a, *args[k + 1:], act=act)).sum()
        _close(got, _differences(f, args[k]))


@pytest.mark.parametrize("kind", ["rbf", "matern12", "matern32", "matern52"])
@pytest.mark.parametrize("ard", [False, True])
def test_input_gradient(rng, kind, ard):
    X = rng.normal(size=(6, 3))
    params = np.array([0.8, 1.1, 0.9, 1.3] if ard else [0.9, 1.3])
    L, R = rng.normal(size=(2, 6)), rng.normal(size=(2, 6))
    got = ol.input_gradient(kind, ard, X, params, L, R)
    _close(got, _differences(lambda a: (ol.kernel(kind, ard, a, params) * (L.T @ R)).sum(), X))


def test_philox_known_answers():
    """The generator authors' published vectors for Philox4x32-10."""
    assert ol.philox(0, 0) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    ones = (1 << 128) - 1
    assert ol.philox(ones, (1 << 64) - 1) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


def test_dropout_keeps_its_share():
    f = ol.dropout_factor((40, 100), 0.25, 7)
    kept = (f > 0).mean()
    assert abs(kept - 0.75) < 5 * np.sqrt(0.25 * 0.75 / 4000)
    assert abs(f.mean() - 1.0) < 5 * np.sqrt(0.25 / 0.75 / 4000)
    assert np.array_equal(f.ravel()[11:], ol.dropout_factor(3989, 0.25, 7, offset=11))
