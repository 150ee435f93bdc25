"""The float64 group norm that the kernels are compared with, its gradients against
central differences (truncation 1e-10, rounding 1e-11 of the function's size)."""

import numpy as np
import pytest

from oracle import layers as ol

STEP, TOL = 1e-5, 2e-7


def _differences(f, a):
    out = np.zeros_like(a)
    for i in np.ndindex(a.shape):
        p, m = a.copy(), a.copy()
        p[i] += STEP
        m[i] -= STEP
        out[i] = (f(p) - f(m)) / (2 * STEP)
    return out


@pytest.mark.parametrize("act", [None, "silu", "gelu", "sigmoid", "relu"])
@pytest.mark.parametrize("shape, groups", [((3, 4, 6), 2), ((2, 6), 3), ((2, 5, 4), 4)])
def test_gradients(rng, act, shape, groups):
    x, w, b = rng.normal(size=shape), rng.normal(size=shape[-1]), rng.normal(size=shape[-1])
    dy = rng.normal(size=shape)
    args = [x, w, b]
    for k, got in enumerate(ol.group_norm_backward(dy, x, groups, w, b, act)):
        def f(a, k=k):
            x, w, b = (*args[:k], a, *args[k + 1:])
            return (dy * ol.group_norm(x, groups, w, b, act)).sum()
        want = _differences(f, args[k])
        assert np.linalg.norm(got - want) <= TOL * (1.0 + np.linalg.norm(want))


def test_one_group_of_one_position_is_layer_norm(rng):
    x, w, b = rng.normal(size=(5, 12)), rng.normal(size=12), rng.normal(size=12)
    assert np.allclose(ol.group_norm(x, 1, w, b), ol.layer_norm(x, w, b), atol=1e-14)
