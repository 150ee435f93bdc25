"""What the group norm's C entries accept, on the host (no device work)."""

import ctypes as C

import pytest

from mojogp_amd import _lib

F32, BF16 = 0, 1
BASE = 1 << 24  # an address that no call gets to read


def _args(**kw):
    a = _lib.GroupNorm(F32, F32, -1, 1e-5, 3, 4, 8, 2, BASE, 8, None, None)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _bytes(a, backward=0):
    nbytes = C.c_int64(0)
    _lib.call("mgp_group_norm_workspace", C.byref(a), backward, C.byref(nbytes))
    return nbytes.value


@pytest.mark.parametrize("kw, what", [
    ({"type": 7}, "element type"), ({"param_type": BF16}, "weight and bias"),
    ({"activation": 4}, "activation"), ({"activation": -2}, "activation"),
    ({"eps": -1.0}, "eps"), ({"eps": float("inf")}, "eps"), ({"samples": -1}, "samples"),
    ({"positions": 1 << 31}, "samples"), ({"samples": 1 << 20, "positions": 1 << 11}, "samples"),
    ({"channels": 0}, "channels"), ({"channels": (1 << 24) + 1}, "channels"),
    ({"groups": 3}, "multiple"), ({"groups": 0}, "multiple"), ({"x": None}, "null device array x"),
    ({"x_stride": 7}, "row stride of x"),
])
def test_arguments_are_refused(kw, what):
    for backward in (0, 1):
        with pytest.raises(_lib.NativeCallError, match=what):
            _bytes(_args(**kw), backward)


def test_workspaces():
    """None for samples that a workgroup holds, forward; partial sums otherwise, at most
    about 2048 stretches."""
    assert _bytes(_args()) == 0
    assert _bytes(_args(), 1) == 256
    big = _args(samples=32, positions=4096, channels=512, groups=32, x_stride=512)
    for backward in (0, 1):
        assert 32 * 512 * 8 < _bytes(big, backward) <= 2048 * 512 * 8 + 32 * 32 * 8
    assert _bytes(_args(samples=1, positions=(1 << 31) - 1, channels=1 << 24, groups=1 << 24,
                        x_stride=1 << 24)) > 0


def test_results_that_share_memory():
    a = _args()
    stats = BASE + 8192

    def forward(y, y_stride=8, s=None):
        _lib.call("mgp_group_norm_device", C.byref(a), y, y_stride, s, None, 0, None)

    for y, kw in ((BASE + 4, {}), (BASE, {"y_stride": 16}), (BASE + 4096, {"s": BASE + 8}),
                  (BASE + 4096, {"s": BASE + 4096 + 376})):
        with pytest.raises(_lib.NativeCallError, match="shares memory with"):
            forward(y, **kw)
    with pytest.raises(_lib.NativeCallError, match="aligned"):
        forward(BASE + 4096, s=stats + 4)

    def backward(dx, dw=None, db=None, ws=BASE + 16384):
        _lib.call("mgp_group_norm_backward_device", C.byref(a), BASE + 4096, 8, stats, dx, 8, dw,
                  db, ws, 1 << 20, None)

    for args, what in (((BASE + 4,), "dx shares memory with x"),
                       ((BASE + 4096 + 32,), "dx shares memory with dy"),
                       ((None, BASE + 4096), "dweight shares memory with dy"),
                       ((None, stats), "dweight shares memory with stats"),
                       ((None, BASE + 65536, BASE + 65536 + 16), "dweight shares memory with dbias"),
                       ((BASE + 65536, BASE + 65536 + 64), "dweight shares memory with dx")):
        with pytest.raises(_lib.NativeCallError, match=what):
            backward(*args)
    with pytest.raises(_lib.NativeCallError, match="256-byte"):
        backward(None, BASE + 65536, ws=BASE + 16384 + 8)


@pytest.mark.parametrize("samples", [1000, 100000, 1 << 22, (1 << 31) - 1])
@pytest.mark.parametrize("positions, channels, groups, kind", [
    (1, 256, 32, BF16), (1, 5000, 8, BF16), (1, 3776, 16, F32), (2, 8192, 4, BF16),
    (4, 16384, 64, F32), (1, 1 << 20, 1 << 10, BF16)])
def test_partial_sums_of_the_parameters_do_not_grow_with_the_samples(samples, positions, channels,
                                                                     groups, kind):
    """Of samples in registers, whole or in blocks of groups: at most 1024 rows."""
    a = _args(type=kind, param_type=kind, samples=min(samples, ((1 << 31) - 1) // positions),
              positions=positions, channels=channels, groups=groups, x_stride=channels)
    assert _bytes(a) == 0
    assert 0 < _bytes(a, 1) <= 1024 * channels * 8 + 256
