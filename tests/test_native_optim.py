"""What the AdamW entry points accept, on the host (no device work)."""

import ctypes as C

import pytest
import torch

from mojogp_amd import _lib, optim

F32, BF16 = 0, 1
BASE = 1 << 24  # addresses that no call gets to read


def _args(sizes, kind=F32, bits=32, master=0, at=None, decay=0.0, **kw):
    at = at or [BASE + 65536 * i for i in range(len(sizes))]
    tensors = (_lib.AdamWTensor * len(sizes))(*[(a, n, decay) for a, n in zip(at, sizes)])
    state = {"exp_avg": 1 << 32, "exp_avg_sq": 2 << 32, "exp_avg_scale": 3 << 32,
             "exp_avg_sq_scale": 4 << 32, "master": 5 << 32, "table": 6 << 32}
    a = _lib.AdamW(type=kind, bits=bits, master_copies=master, count=len(sizes), tensors=tensors,
                   beta1=0.9, beta2=0.999, eps=1e-8, **state)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _layout(a):
    values, nbytes = C.c_int64(0), C.c_int64(0)
    _lib.call("mgp_adamw_layout", C.byref(a), C.byref(values), C.byref(nbytes))
    return values.value, nbytes.value


def _create(a):
    host = (C.c_char * _layout(a)[1])()
    plan = C.c_void_p()
    _lib.call("mgp_adamw_create", C.byref(a), host, len(host), C.byref(plan))
    return plan, host


def _step(plan, count, grads=None, **kw):
    s = _lib.AdamWStep(grads=(C.c_void_p * count)(*(grads or [None] * count)), grad_type=F32,
                       grad_scale=1.0, max_norm=1.0, step=1, rate=1e-3)
    for k, v in kw.items():
        setattr(s, k, v)
    _lib.call("mgp_adamw_step_device", plan, C.byref(s), None, 0, None)


def test_layout_and_table():
    """Every tensor's values start at a multiple of 256; 32 bytes a tensor and 8 for
    each 2048 values."""
    a = _args([1, 256, 257, 0, 5000])
    assert _layout(a) == (256 + 256 + 512 + 5120, 5 * 32 + (1 + 1 + 1 + 0 + 3) * 8)
    plan, host = _create(a)
    import struct
    raw = bytes(host)
    rows = [struct.unpack_from("qqqff", raw, 32 * i) for i in range(5)]
    assert [r[1] for r in rows] == [1, 256, 257, 0, 5000]
    assert [r[2] for r in rows] == [0, 256, 512, 1024, 1024]
    chunks = [struct.unpack_from("II", raw, 160 + 8 * i) for i in range(6)]
    assert chunks == [(0, 0), (1, 0), (2, 0), (4, 0), (4, 1), (4, 2)]
    _lib.call("mgp_adamw_destroy", plan)
    with pytest.raises(_lib.NativeCallError, match="unknown or destroyed"):
        _lib.call("mgp_adamw_destroy", plan)
    with pytest.raises(_lib.NativeCallError, match="unknown or destroyed"):
        _step(plan, 5)


@pytest.mark.parametrize("kw, what", [
    ({"bits": 16}, "32 or 8 bits"), ({"beta1": 1.0}, "decay rates"), ({"beta2": -0.1}, "decay"),
    ({"eps": 0.0}, "eps"), ({"eps": float("nan")}, "eps"), ({"master": 1, "kind": F32}, "master"),
    ({"kind": 7}, "element type"), ({"decay": -1.0}, "weight decay"),
    ({"decay": float("inf")}, "weight decay"), ({"count": 0}, "count"),
])
def test_arguments_are_refused(kw, what):
    master = kw.pop("master", 0)
    with pytest.raises(_lib.NativeCallError, match=what):
        _layout(_args([10], master=0 if master is None else master, **kw))


def test_tensors_are_refused():
    for sizes in ([-1], [1 << 40], [1 << 34] * 3):
        with pytest.raises(_lib.NativeCallError, match="too large|too many"):
            _layout(_args(sizes))
    with pytest.raises(_lib.NativeCallError, match="null parameter"):
        _layout(_args([4], at=[None]))
    # the same tensor twice, one inside another, and on the states
    for at in ([BASE, BASE], [BASE, BASE + 396], [BASE, 1 << 32], [BASE, (6 << 32) + 8]):
        with pytest.raises(_lib.NativeCallError, match="shares memory with"):
            _create(_args([100, 50], at=at))
    plan, _ = _create(_args([100, 50], at=[BASE, BASE + 400]))
    _lib.call("mgp_adamw_destroy", plan)


def test_steps_are_refused():
    a = _args([100, 50])
    plan, _ = _create(a)
    try:
        for grads, what in (([BASE + 396, None], "a parameter"), ([None, 1 << 32], "the states"),
                            ([(2 << 32) - 4, None], "the states"), ([BASE - 396, None], "a parameter")):
            with pytest.raises(_lib.NativeCallError, match="a gradient shares memory with " + what):
                _step(plan, 2, grads)
        for kw, what in (({"step": 0}, "step"), ({"rate": -1.0}, "rate"),
                         ({"rate": float("nan")}, "rate"), ({"grad_scale": 0.0}, "scale"),
                         ({"grad_type": BF16}, "gradients must be"), ({"form_norm": 1}, "workspace"),
                         ({"form_norm": 1, "max_norm": 0.0}, "max_norm"),
                         ({"step_device": BASE}, "workspace")):
            with pytest.raises(_lib.NativeCallError, match=what):
                _step(plan, 2, **kw)
    finally:
        _lib.call("mgp_adamw_destroy", plan)


def test_what_a_step_writes_shares_no_memory():
    """The workspace and the norm with the gradients, the step, the rate and each other."""
    plan, _ = _create(_args([100, 50]))
    ws = 7 << 32
    try:
        for grads, kw, what in (
                ([None, ws - 196], {}, "a gradient shares memory with the workspace"),
                ([None, BASE - 400], {"norm": BASE - 204}, "a gradient shares memory with norm"),
                ([None, None], {"norm": ws + 8}, "norm shares memory with the workspace"),
                ([None, None], {"norm": BASE - 64, "step_device": BASE - 64},
                 "step shares memory with norm"),
                ([None, None], {"rate_device": ws + 252}, "rate shares memory with the workspace")):
            s = _lib.AdamWStep(grads=(C.c_void_p * 2)(*grads), grad_type=F32, grad_scale=1.0,
                               form_norm=1, max_norm=1.0, step=1, rate=1e-3)
            for k, v in kw.items():
                setattr(s, k, v)
            nbytes = C.c_int64(0)
            _lib.call("mgp_adamw_workspace", plan, C.byref(s), C.byref(nbytes))
            with pytest.raises(_lib.NativeCallError, match=what):
                _lib.call("mgp_adamw_step_device", plan, C.byref(s), ws, nbytes.value, None)
    finally:
        _lib.call("mgp_adamw_destroy", plan)
    plan, _ = _create(_args([100], bits=8))
    try:
        with pytest.raises(_lib.NativeCallError, match="the results share memory"):
            _lib.call("mgp_adamw_values_device", plan, 8 << 32, (8 << 32) + 1020, None)
    finally:
        _lib.call("mgp_adamw_destroy", plan)


def test_python_entry_refuses_what_is_on_the_host():
    with pytest.raises(ValueError, match="device tensors"):
        optim.AdamW([torch.zeros(4)])
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        optim.AdamW([torch.zeros(4, dtype=torch.float64)])
    with pytest.raises(ValueError, match="at least one"):
        optim.AdamW([])
