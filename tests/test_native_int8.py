"""What the 8-bit layers' C entries accept, on the host (no device work)."""

import ctypes as C

import pytest

from mojogp_amd import _lib

F32 = 0
BASE = 1 << 24  # addresses that no call gets to read


def _args(**kw):
    a = _lib.Int8Layer(F32, -1, 20, 24, 8, BASE, 24, BASE + (1 << 16), None, 32, BASE + (1 << 17),
                       None, None, None)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _bytes(a):
    nbytes = C.c_int64(0)
    _lib.call("mgp_int8_layer_workspace", C.byref(a), C.byref(nbytes))
    return nbytes.value


def test_workspace_holds_codes_and_scales():
    assert _bytes(_args()) == 768 + 256  # 20 rows of 32 bytes, 20 floats
    assert _bytes(_args(rows=16)) == 0   # few rows are quantised where they are used
    assert _bytes(_args(rows=0, x=None)) == 0


@pytest.mark.parametrize("kw, what", [
    ({"type": 3}, "element type"), ({"activation": 9}, "activation"),
    ({"activation": -1, "w_up": BASE, "s_up": BASE}, "activation"), ({"rows": -1}, "rows"),
    ({"width": 0}, "width"), ({"width": 131073, "x_stride": 131073, "w_stride": 131088}, "131072"),
    ({"hidden": 0}, "hidden"), ({"x": None}, "null device array x"), ({"x_stride": 23}, "row stride"),
    ({"w_gate": None}, "null device array w_gate"), ({"w_gate": BASE + 8}, "16-byte"),
    ({"w_stride": 24}, "16-byte"), ({"w_stride": 16}, "16-byte"), ({"w_stride": 1 << 23}, "8 MB"),
    ({"s_gate": None}, "null scales"), ({"s_up": BASE}, "null scales"),
    ({"w_up": BASE, "activation": 0}, "null scales"),
    ({"w_up": BASE + 4, "s_up": BASE, "activation": 0}, "16-byte"),
])
def test_arguments_are_refused(kw, what):
    with pytest.raises(_lib.NativeCallError, match=what):
        _bytes(_args(**kw))


def test_results_that_share_memory():
    a = _args(b_gate=BASE + (1 << 18))
    for y, what in ((BASE, "x"), (BASE + 1916, "x"), (BASE + (1 << 16) + 252, "w_gate"),
                    (BASE + (1 << 17), "s_gate"), (BASE + (1 << 18) + 28, "b_gate")):
        with pytest.raises(_lib.NativeCallError, match="y shares memory with " + what):
            _lib.call("mgp_int8_layer_device", C.byref(a), y, 8, None, 0, None)
    with pytest.raises(_lib.NativeCallError, match="workspace of 0 bytes"):
        _lib.call("mgp_int8_layer_device", C.byref(a), BASE + (1 << 20), 8, None, 0, None)


def test_quantize_refuses():
    def call(codes, stride=16, scales=BASE + (1 << 17), width=10, rows=4):
        _lib.call("mgp_int8_quantize_device", F32, BASE, width, rows, width, codes, stride, scales,
                  None)

    far = BASE + (1 << 16)
    for kw, what in (({"codes": far + 4}, "16-byte"), ({"codes": far, "stride": 12}, "16-byte"),
                     ({"codes": far, "stride": 16, "width": 17}, "16-byte"),
                     ({"codes": None}, "null device array codes"),
                     ({"codes": far, "scales": None}, "null scales"),
                     ({"codes": far, "width": 131073, "stride": 131088}, "131072"),
                     ({"codes": BASE + 144}, "codes shares memory with x"),
                     ({"codes": far, "scales": BASE + 8}, "scales shares memory with x"),
                     ({"codes": far, "scales": far + 60}, "codes shares memory with scales")):
        with pytest.raises(_lib.NativeCallError, match=what):
            call(**kw)
