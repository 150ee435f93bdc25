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
