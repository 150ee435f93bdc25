"""What the layers' C entry points accept, on the host (no device work)."""

import ctypes as C

import pytest

from mojogp_amd import _lib

F32, BF16, F16 = 0, 1, 2


def _workspace(kind, rows, width, hidden, backward):
    a = _lib.GatedLayer(kind, 0, rows, width, hidden, 1 << 20, width, 1 << 20, width, 1 << 20,
                        width, None, None)
    nbytes = C.c_int64(0)
    _lib.call("mgp_gated_layer_workspace", C.byref(a), backward, C.byref(nbytes))
    return nbytes.value


@pytest.mark.parametrize("kind, rows, most", [(F32, 200, 699040), (F32, 5, 699040),
                                              (BF16, 200, 2097144), (BF16, 128, 1048568),
                                              (F16, 200, 2097144)])
def test_hidden_width_within_the_loads_offsets(kind, rows, most):
    """The products form a row's offset in 31 bits over the 256 rows of a tile: rows
    of [dg | du] of 8 MB and more would be read from wrong addresses."""
    assert _workspace(kind, rows, 64, most, 1) > rows * most * 4
    for hidden in (most + 1, 1 << 23, 1 << 24):
        with pytest.raises(_lib.NativeCallError, match="hidden width"):
            _workspace(kind, rows, 64, hidden, 1)


@pytest.mark.parametrize("kind, most", [(F32, 1398080), (BF16, 4194296), (F16, 4194296)])
def test_width_within_the_loads_offsets(kind, most):
    for backward in (0, 1):
        _workspace(kind, 70, most, 16384, backward)
        with pytest.raises(_lib.NativeCallError, match="the width"):
            _workspace(kind, 70, most + 1, 16384, backward)
    # few rows and columns go without the products
    assert _workspace(kind, 1, 1 << 24, 64, 0) == 0


BASE = 1 << 24  # an address that no call gets to read


def _norm(x, y, rows=4, width=8, x_stride=8, y_stride=8, stats=None, weight=None):
    a = _lib.LayerNorm(F32, F32, 1e-5, rows, width, x, x_stride, weight, None)
    _lib.call("mgp_layer_norm_device", C.byref(a), y, y_stride, stats, None)


@pytest.mark.parametrize("x, y, kw", [
    (BASE, BASE + 4, {}), (BASE, BASE + 32, {}), (BASE + 32, BASE, {}),
    (BASE, BASE, {"y_stride": 16}),
    (BASE, BASE + 28, {"x_stride": 16, "y_stride": 16}),   # a column in common
    (BASE, BASE + 3 * 64 + 28, {"x_stride": 16, "y_stride": 16}),  # in one row
    (BASE, BASE + 48, {"x_stride": 16, "y_stride": 16}),   # runs on into the next row
    (BASE, BASE + 4096, {"stats": BASE + 8}), (BASE, BASE + 4096, {"stats": BASE + 4096 + 120}),
    (BASE, BASE + 4096, {"weight": BASE + 4096 + 120}),
])
def test_layer_norm_refuses_results_that_share_memory(x, y, kw):
    with pytest.raises(_lib.NativeCallError, match="shares memory with"):
        _norm(x, y, **kw)


def test_layer_norm_backward_refuses_results_that_share_memory():
    a = _lib.LayerNorm(F32, F32, 1e-5, 4, 8, BASE, 8, None, None)
    stats, ws = BASE + 8192, BASE + 16384
    for dx, dw, what in ((BASE + 4, None, "dx shares memory with x"),
                         (BASE + 4096 + 96, None, "dx shares memory with dy"),
                         (None, BASE + 4096 + 64, "dweight shares memory with dy"),
                         (None, stats, "dweight shares memory with stats")):
        with pytest.raises(_lib.NativeCallError, match=what):
            _lib.call("mgp_layer_norm_backward_device", C.byref(a), BASE + 4096, 8, stats, dx, 8,
                      dw, None, ws, 1 << 20, None)


def test_dropout_refuses_results_that_share_memory():
    for y, residual in ((BASE + 4, None), (BASE + 4096, BASE + 4096 + 4), (BASE - 4, None)):
        with pytest.raises(_lib.NativeCallError, match="y shares memory with"):
            _lib.call("mgp_dropout_device", F32, BASE, 8, 4, 8, 0.1, 1, 0, residual, 8, y, 8, None)


def test_gated_layer_refuses_results_that_share_memory():
    x, wg, wu, bg, dh = (BASE + k * 4096 for k in range(5))
    a = _lib.GatedLayer(F32, 0, 4, 8, 8, x, 8, wg, 8, wu, 8, bg, None)
    for h, what in ((x, "x"), (x + 124, "x"), (wg, "w_gate"), (wu + 252, "w_up"), (bg, "b_gate")):
        with pytest.raises(_lib.NativeCallError, match="h shares memory with " + what):
            _lib.call("mgp_gated_layer_device", C.byref(a), h, 8, None, 0, None)
    free = BASE + (1 << 20)
    for k, name in enumerate(("dx", "dw_gate", "dw_up", "db_gate", "db_up")):
        for at, what in ((x, "x"), (dh, "dh"), (bg, "b_gate")):
            out = [free + 4096 * j for j in range(5)]
            out[k] = at
            with pytest.raises(_lib.NativeCallError, match=f"{name} shares memory with {what}"):
                _lib.call("mgp_gated_layer_backward_device", C.byref(a), dh, 8, *out,
                          BASE + (1 << 22), 1 << 22, None)
