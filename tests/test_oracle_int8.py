"""The layers in 8-bit integers that the kernels are compared with."""

import numpy as np

from oracle import layers as ol


def test_rows():
    q, s = ol.int8_rows([[1.0, -2.0, 0.5, 0.0], [0, 0, 0, 0], [127.0, 0.5, 1.5, -2.5],
                         [1e-37, 0, 0, 0]])
    assert q.tolist() == [[64, -127, 32, 0], [0] * 4, [127, 0, 2, -2], [0] * 4]
    assert s[0] == np.float32(2 / 127) and s[1] == 0 and s[2] == 1 and s[3] == 0


def test_layer_is_near_the_product(rng):
    """Each side is rounded by at most half a step of its rows' largest value / 127."""
    x, w, b = rng.normal(size=(20, 64)), rng.normal(size=(30, 64)), rng.normal(size=30)
    y, size = ol.int8_layer(x, w, b)
    step = np.abs(x).max(axis=1)[:, None] / 254, np.abs(w).max(axis=1) / 254
    most = (step[0] * np.abs(w).sum(axis=1) + step[1] * np.abs(x).sum(axis=1)[:, None]
            + 64 * step[0] * step[1]) * 1.01
    assert (np.abs(y - (x @ w.T + b)) <= most).all()
    assert np.allclose(size, np.abs(y - b))
    gated, _ = ol.int8_layer(x, w, b, w[::-1], b, "silu")
    g, u = ol.int8_layer(x, w, b)[0], ol.int8_layer(x, w[::-1], b)[0]
    assert np.allclose(gated, ol.activate("silu", g)[0] * u)
