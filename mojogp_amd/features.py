"""The layers of a deep kernel: learned features in front of a Gaussian process.

    h = gated_layer(x, w_gate, w_up, b_gate, b_up)      # act(x Wg^T + bg) * (x Wu^T + bu)
    y, saved = layer_norm(h, weight, bias, save=True)
    z = dropout(y, 0.1, seed, offset=step * y.numel())

and their gradients (``gated_layer_backward``, ``layer_norm_backward``,
``dropout_backward``).  The gradient that enters at the top is
``NativeProvider.input_gradient_device``: that of the marginal likelihood with
respect to the kernel's points.

Arrays are device tensors of the calling program (float32, bfloat16 or
float16, unit stride along the last dimension, leading dimensions that collapse
to one row stride).  Their addresses go to the library's kernels; torch is not
imported here and computes nothing, it provides the arrays, the memory of the
results and the current stream, on which every call runs asynchronously.  The
calls are explicit forward and backward passes and take no part in autograd.
"""

from __future__ import annotations

import ctypes as C
import sys
from typing import NamedTuple

from . import _lib

ACTIVATIONS = {"silu": 0, "gelu": 1, "sigmoid": 2, "relu": 3}

_MAX_DRAWS = 1 << 64


class GatedGradients(NamedTuple):
    """What gated_layer_backward returns; None where it was not asked for."""
    dx: object
    dw_gate: object
    dw_up: object
    db_gate: object
    db_up: object


_types: dict = {}


def _elem(a, name):
    """Element type code of a tensor; torch is loaded if there is one."""
    if not _types:
        torch = sys.modules.get("torch")
        if torch is not None:
            _types.update({torch.float32: 0, torch.bfloat16: 1, torch.float16: 2})
    code = _types.get(getattr(a, "dtype", None))
    if code is None:
        raise TypeError(f"{name} must be a float32, bfloat16 or float16 device tensor, got "
                        f"{getattr(a, 'dtype', type(a).__name__)}")
    return code


def _first(a, name):
    """(element type, device index, stream) of a call from its first array."""
    code = _elem(a, name)
    if not a.is_cuda:
        raise ValueError(f"{name} must be a device tensor, got one on {a.device}")
    cuda = sys.modules["torch"].cuda
    index = a.device.index
    if index != cuda.current_device():
        raise ValueError(f"{name} is on device {index}, the current device is "
                         f"{cuda.current_device()}")
    return code, index, cuda.current_stream(index).cuda_stream


def _rows(a, name, code, index, shape=None):
    """(address, rows, width, row stride) of an array as a matrix of rows."""
    if _elem(a, name) != code:
        raise TypeError(f"{name} must have the element type of the first array, got {a.dtype}")
    if not a.is_cuda or a.device.index != index:
        raise ValueError(f"{name} must be on device {index}, got {a.device}")
    if shape is not None and a.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(a.shape)}")
    dims = a.dim()
    if dims == 0:
        raise ValueError(f"{name} must have at least one dimension")
    width = a.shape[-1]
    if width == 0:
        raise ValueError(f"{name} must have at least one column")
    if width > 1 and a.stride(-1) != 1:
        raise ValueError(f"{name} must have unit stride along its last dimension, got strides "
                         f"{a.stride()}")
    if dims == 1:
        return a.data_ptr(), 1, width, width
    if dims == 2:
        rows, stride = a.shape[0], a.stride(0)
    else:
        rows, stride = _collapse(a, name)
    if rows <= 1:
        stride = width
    elif stride < width:
        raise ValueError(f"{name} has rows that overlap (stride {stride}, width {width})")
    return a.data_ptr(), rows, width, stride


def _collapse(a, name):
    """Rows and row stride of more than two dimensions."""
    rows, stride = 1, a.shape[-1]
    for size, step in zip(reversed(a.shape[:-1]), reversed(a.stride()[:-1])):
        if size == 1:
            continue
        if rows == 1:
            stride = step
        elif step != rows * stride:
            raise ValueError(f"the leading dimensions of {name} do not collapse to rows of one "
                             f"stride (shape {tuple(a.shape)}, strides {a.stride()})")
        rows *= size
    return rows, stride


def _vector(a, name, width, code, index, also=None):
    """Address of a contiguous [width] vector, or None."""
    if a is None:
        return None
    got = _elem(a, name)
    if got != code and got != also:
        raise TypeError(f"{name} has element type {a.dtype}, which does not fit the other arrays")
    if not a.is_cuda or a.device.index != index:
        raise ValueError(f"{name} must be on device {index}, got {a.device}")
    if a.dim() != 1 or a.shape[0] != width:
        raise ValueError(f"{name} must have shape ({width},), got {tuple(a.shape)}")
    if width > 1 and a.stride(0) != 1:
        raise ValueError(f"{name} must be contiguous")
    return a.data_ptr()


def _result(a, name, like, code, index):
    """A given result array (checked against `like`), or a new contiguous one."""
    if a is None:
        return like.new_empty(like.shape)
    _rows(a, name, code, index, like.shape)
    return a


def _workspace(like, nbytes):
    return like.new_empty((nbytes,), dtype=sys.modules["torch"].uint8) if nbytes else None


def _address(a):
    return None if a is None else a.data_ptr()


# ---------------------------------------------------------------- layer norm

def _norm_args(x, weight, bias, eps):
    code, index, stream = _first(x, "x")
    px, rows, width, stride = _rows(x, "x", code, index)
    pw = _vector(weight, "weight", width, code, index, also=0)
    pb = _vector(bias, "bias", width, code, index, also=0)
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError("weight and bias must have one element type")
    given = weight if weight is not None else bias
    ptype = code if given is None else _types[given.dtype]
    return _lib.LayerNorm(code, ptype, eps, rows, width, px, stride, pw, pb), index, stream


def layer_norm(x, weight=None, bias=None, eps=1e-5, *, save=False, out=None):
    """Layer norm over the last dimension: ``(x - mean) / sqrt(var + eps) * weight + bias``.

    weight and bias ([width], of x's type or float32) may be None.  With
    ``save=True`` returns ``(y, saved)``, ``saved`` being what the backward
    pass takes (mean and reciprocal deviation of every row, float32)."""
    a, index, stream = _norm_args(x, weight, bias, eps)
    y = _result(out, "out", x, a.type, index)
    py, _, _, stride = _rows(y, "out", a.type, index)
    stats = x.new_empty((a.rows, 2), dtype=sys.modules["torch"].float32) if save else None
    _lib.call("mgp_layer_norm_device", C.byref(a), py, stride, _address(stats), stream)
    return (y, stats) if save else y


def layer_norm_backward(dy, x, weight, saved, *, bias=True):
    """Gradients ``(dx, dweight, dbias)`` of ``layer_norm(x, weight, bias)``.

    dweight and dbias have weight's type (x's where weight is None; dweight is
    then None).  ``bias=False``: the layer has none, dbias is None."""
    a, index, stream = _norm_args(x, weight, None, 0.0)
    pdy, _, _, dy_stride = _rows(dy, "dy", a.type, index, x.shape)
    if saved is None or tuple(saved.shape) != (a.rows, 2) or _elem(saved, "saved") != 0 \
            or not saved.is_contiguous() or saved.device != x.device:
        raise ValueError("saved must be what layer_norm(..., save=True) returned for this x")
    dx = x.new_empty(x.shape)
    params = x if weight is None else weight
    dweight = None if weight is None else params.new_empty((a.width,))
    dbias = params.new_empty((a.width,)) if bias else None
    nbytes = C.c_int64(0)
    if dweight is not None or dbias is not None:
        _lib.call("mgp_layer_norm_backward_workspace", C.byref(a), C.byref(nbytes))
    ws = _workspace(x, nbytes.value)
    _lib.call("mgp_layer_norm_backward_device", C.byref(a), pdy, dy_stride, saved.data_ptr(),
              dx.data_ptr(), a.width, _address(dweight), _address(dbias), _address(ws),
              nbytes.value, stream)
    return dx, dweight, dbias


# ---------------------------------------------------------------- dropout

def _dropout(x, name, rate, seed, offset, residual, out):
    code, index, stream = _first(x, name)
    px, rows, width, stride = _rows(x, name, code, index)
    pr, r_stride = None, 0
    if residual is not None:
        pr, _, _, r_stride = _rows(residual, "residual", code, index, x.shape)
    if not 0 <= seed < _MAX_DRAWS or not 0 <= offset < _MAX_DRAWS:
        raise ValueError("seed and offset must be in [0, 2^64)")
    y = _result(out, "out", x, code, index)
    py, _, _, y_stride = _rows(y, "out", code, index)
    _lib.call("mgp_dropout_device", code, px, stride, rows, width, rate, seed, offset, pr,
              r_stride, py, y_stride, stream)
    return y


def dropout(x, rate, seed, *, offset=0, residual=None, out=None):
    """``residual + x * keep / (1 - rate)`` with a mask that is never stored.

    Whether element i (row-major) of x is kept is a function of ``seed`` and the
    draw number ``offset + i`` alone, so that ``dropout_backward`` with the same
    seed and offset draws the same mask; the next call's offset is this one's
    plus ``x.numel()`` (multiples of 8 are fastest).  The rate in effect is
    ``rate`` rounded to a multiple of 2^-16.  ``out`` may be x or residual."""
    return _dropout(x, "x", rate, seed, offset, residual, out)


def dropout_backward(dy, rate, seed, *, offset=0, out=None):
    """Gradient of ``dropout`` with respect to x (that of residual is dy)."""
    return _dropout(dy, "dy", rate, seed, offset, None, out)


# ---------------------------------------------------------------- gated layer

def _gated_args(x, w_gate, w_up, b_gate, b_up, activation):
    code, index, stream = _first(x, "x")
    try:
        act = ACTIVATIONS[activation]
    except (KeyError, TypeError):
        raise ValueError(f"unknown activation {activation!r}; one of {sorted(ACTIVATIONS)}") \
            from None
    px, rows, width, stride = _rows(x, "x", code, index)
    if w_gate.dim() != 2 or w_gate.shape[1] != width:
        raise ValueError(f"w_gate must have shape (hidden, {width}), got {tuple(w_gate.shape)}")
    pg, hidden, _, g_stride = _rows(w_gate, "w_gate", code, index)
    if hidden == 0:
        raise ValueError("w_gate must have at least one row")
    pu, _, _, u_stride = _rows(w_up, "w_up", code, index, w_gate.shape)
    bg = _vector(b_gate, "b_gate", hidden, code, index)
    bu = _vector(b_up, "b_up", hidden, code, index)
    return _lib.GatedLayer(code, act, rows, width, hidden, px, stride, pg, g_stride, pu, u_stride,
                           bg, bu), index, stream


def _gated_workspace(a, x, backward):
    nbytes = C.c_int64(0)
    _lib.call("mgp_gated_layer_workspace", C.byref(a), backward, C.byref(nbytes))
    return _workspace(x, nbytes.value), nbytes.value


def gated_layer(x, w_gate, w_up, b_gate=None, b_up=None, *, activation="silu", out=None):
    """``act(x w_gate^T + b_gate) * (x w_up^T + b_up)`` in one kernel.

    x [..., width], weights [hidden, width], biases [hidden] or None, all of one
    element type; result [..., hidden].  activation: "silu", "gelu" (with the
    normal distribution's exact integral), "sigmoid" or "relu"."""
    a, index, stream = _gated_args(x, w_gate, w_up, b_gate, b_up, activation)
    shape = (*x.shape[:-1], a.hidden)
    if out is None:
        out = x.new_empty(shape)
    elif tuple(out.shape) != shape:
        raise ValueError(f"out must have shape {shape}, got {tuple(out.shape)}")
    ph, _, _, h_stride = _rows(out, "out", a.type, index)
    ws, nbytes = _gated_workspace(a, x, 0)
    _lib.call("mgp_gated_layer_device", C.byref(a), ph, h_stride, _address(ws), nbytes, stream)
    return out


def gated_layer_backward(dh, x, w_gate, w_up, b_gate=None, b_up=None, *, activation="silu",
                         need_dx=True, need_dw=True):
    """Gradients of ``gated_layer`` as ``GatedGradients(dx, dw_gate, dw_up, db_gate, db_up)``.

    The projections are formed again from x: nothing is kept between the
    passes.  ``need_dx=False`` (the first layer, whose x is data) and
    ``need_dw=False`` leave those products out."""
    a, index, stream = _gated_args(x, w_gate, w_up, b_gate, b_up, activation)
    if tuple(dh.shape) != (*x.shape[:-1], a.hidden):
        raise ValueError(f"dh must have shape {(*x.shape[:-1], a.hidden)}, got {tuple(dh.shape)}")
    pdh, _, _, dh_stride = _rows(dh, "dh", a.type, index)
    g = GatedGradients(
        x.new_empty(x.shape) if need_dx else None,
        x.new_empty((a.hidden, a.width)) if need_dw else None,
        x.new_empty((a.hidden, a.width)) if need_dw else None,
        x.new_empty((a.hidden,)) if b_gate is not None else None,
        x.new_empty((a.hidden,)) if b_up is not None else None)
    ws, nbytes = _gated_workspace(a, x, 1)
    _lib.call("mgp_gated_layer_backward_device", C.byref(a), pdh, dh_stride,
              *(_address(t) for t in g), _address(ws), nbytes, stream)
    return g
