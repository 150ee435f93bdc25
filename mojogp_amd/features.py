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
calls are explicit forward and backward passes and take no part in autograd: an
array that requires a gradient is refused unless torch.no_grad() says that none is
recorded.
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


_types: dict = {}  # torch's element types and this library's codes


def _torch():
    """torch, which a program that holds device tensors has loaded."""
    torch = sys.modules.get("torch")
    if torch is None:
        raise TypeError("the arrays must be device tensors of torch")
    if not _types:
        _types.update({torch.float32: 0, torch.bfloat16: 1, torch.float16: 2})
    return torch


def _stream(torch, index):
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)  # without making an object of it
    return raw(index) if raw else torch.cuda.current_stream(index).cuda_stream


def _first(a, name):
    """(element type, its code, device index, stream) of a call from its first array."""
    torch = _torch()
    dtype = getattr(a, "dtype", None)
    code = _types.get(dtype)
    if code is None:
        raise TypeError(f"{name} must be a float32, bfloat16 or float16 device tensor, got "
                        f"{dtype or type(a).__name__}")
    if a.requires_grad:
        _no_graph(name)
    index = a.get_device()
    if index < 0:
        raise ValueError(f"{name} must be a device tensor, got one on {a.device}")
    current = torch.cuda.current_device()
    if index != current:
        raise ValueError(f"{name} is on device {index}, the current device is {current}")
    return dtype, code, index, _stream(torch, index)


def _no_graph(name):
    """These calls record nothing: where a graph is being recorded, it would end here
    without a word."""
    if _torch().is_grad_enabled():
        raise ValueError(f"{name} requires a gradient, which these calls do not record: use "
                         "detach() or torch.no_grad() and the explicit backward passes")


def _check(a, name, dtype, index):
    if getattr(a, "dtype", None) is not dtype:
        raise TypeError(f"{name} must have the element type of the first array ({dtype}), got "
                        f"{getattr(a, 'dtype', type(a).__name__)}")
    if a.requires_grad:
        _no_graph(name)
    if a.get_device() != index:
        raise ValueError(f"{name} must be on device {index}, got {a.device}")


def _rows(a, name, dtype, index, shape=None):
    """(address, rows, width, row stride) of an array as a matrix of rows."""
    _check(a, name, dtype, index)
    got, strides = a.shape, a.stride()
    if shape is not None and got != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(got)}")
    dims = len(got)
    if dims == 2:
        rows, width = got
        stride = strides[0]
    elif dims == 1:
        rows, width, stride = 1, got[0], 0
    elif dims == 0:
        raise ValueError(f"{name} must have at least one dimension")
    else:
        width = got[-1]
        rows, stride = _collapse(got, strides, name)
    if width == 0:
        raise ValueError(f"{name} must have at least one column")
    if strides[-1] != 1 and width > 1:
        raise ValueError(f"{name} must have unit stride along its last dimension, got strides "
                         f"{strides}")
    if rows <= 1:
        stride = width
    elif stride < width:
        raise ValueError(f"{name} has rows that overlap (stride {stride}, width {width})")
    return a.data_ptr(), rows, width, stride


def _collapse(shape, strides, name):
    """Rows and row stride of more than two dimensions."""
    if 0 in shape[:-1]:
        return 0, shape[-1]
    rows, stride = 1, shape[-1]
    for size, step in zip(reversed(shape[:-1]), reversed(strides[:-1])):
        if size == 1:
            continue
        if rows == 1:
            stride = step
        elif step != rows * stride:
            raise ValueError(f"the leading dimensions of {name} do not collapse to rows of one "
                             f"stride (shape {tuple(shape)}, strides {strides})")
        rows *= size
    return rows, stride


def _vector(a, name, width, dtype, index):
    """Address of a contiguous [width] vector, or None."""
    if a is None:
        return None
    _check(a, name, dtype, index)
    if a.shape != (width,):
        raise ValueError(f"{name} must have shape ({width},), got {tuple(a.shape)}")
    if width > 1 and a.stride(0) != 1:
        raise ValueError(f"{name} must be contiguous")
    return a.data_ptr()


def _result(a, name, like, shape, dtype, index):
    """(array, address, row stride) of a given result, checked, or a new one."""
    if a is None:
        a = like.new_empty(shape)
        return a, a.data_ptr(), shape[-1]
    address, _, _, stride = _rows(a, name, dtype, index, shape)
    return a, address, stride


def _workspace(like, nbytes):
    return like.new_empty((nbytes,), dtype=_torch().uint8) if nbytes else None


def _address(a):
    return None if a is None else a.data_ptr()


# ---------------------------------------------------------------- layer norm

def _norm_args(x, weight, bias, eps):
    dtype, code, index, stream = _first(x, "x")
    px, rows, width, stride = _rows(x, "x", dtype, index)
    given = weight if weight is not None else bias
    ptype, pcode = dtype, code
    if given is not None and given.dtype is not dtype:
        ptype, pcode = given.dtype, _types.get(given.dtype)
        if pcode != 0:
            raise TypeError(f"weight and bias must have x's element type or be float32, got "
                            f"{ptype}, which does not fit {dtype}")
    pw = _vector(weight, "weight", width, ptype, index)
    pb = _vector(bias, "bias", width, ptype, index)
    return (_lib.LayerNorm(code, pcode, eps, rows, width, px, stride, pw, pb), dtype, index,
            stream)


def layer_norm(x, weight=None, bias=None, eps=1e-5, *, save=False, out=None):
    """Layer norm over the last dimension: ``(x - mean) / sqrt(var + eps) * weight + bias``.

    weight and bias ([width], of x's type or float32) may be None.  ``out`` may be
    x, but share no memory with it otherwise.  With
    ``save=True`` returns ``(y, saved)``, ``saved`` being what the backward
    pass takes (mean and reciprocal deviation of every row, float32)."""
    a, dtype, index, stream = _norm_args(x, weight, bias, eps)
    y, py, stride = _result(out, "out", x, x.shape, dtype, index)
    stats = x.new_empty((a.rows, 2), dtype=_torch().float32) if save else None
    _lib.call("mgp_layer_norm_device", C.byref(a), py, stride, _address(stats), stream)
    return (y, stats) if save else y


def layer_norm_backward(dy, x, weight, saved, *, bias=True):
    """Gradients ``(dx, dweight, dbias)`` of ``layer_norm(x, weight, bias)``.

    dweight and dbias have weight's type (x's where weight is None; dweight is
    then None).  ``bias=False``: the layer has none, dbias is None."""
    a, dtype, index, stream = _norm_args(x, weight, None, 0.0)
    pdy, _, _, dy_stride = _rows(dy, "dy", dtype, index, x.shape)
    if saved is None or saved.shape != (a.rows, 2) or _types.get(saved.dtype) != 0 \
            or not saved.is_contiguous() or saved.get_device() != index:
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
    dtype, code, index, stream = _first(x, name)
    px, rows, width, stride = _rows(x, name, dtype, index)
    pr, r_stride = None, 0
    if residual is not None:
        pr, _, _, r_stride = _rows(residual, "residual", dtype, index, x.shape)
    if not 0 <= seed < _MAX_DRAWS or not 0 <= offset < _MAX_DRAWS:
        raise ValueError("seed and offset must be in [0, 2^64)")
    y, py, y_stride = _result(out, "out", x, x.shape, dtype, index)
    _lib.call("mgp_dropout_device", code, px, stride, rows, width, rate, seed, offset, pr,
              r_stride, py, y_stride, stream)
    return y


def dropout(x, rate, seed, *, offset=0, residual=None, out=None):
    """``residual + x * keep / (1 - rate)`` with a mask that is never stored.

    Whether element i (row-major) of x is kept is a function of ``seed`` and the
    draw number ``offset + i`` alone, so that ``dropout_backward`` with the same
    seed and offset draws the same mask; the next call's offset is this one's
    plus ``x.numel()`` (multiples of 8 are fastest).  The rate in effect is
    ``rate`` rounded to a multiple of 2^-16.  ``out`` may be x or residual, but share
    no memory with them otherwise."""
    return _dropout(x, "x", rate, seed, offset, residual, out)


def dropout_backward(dy, rate, seed, *, offset=0, out=None):
    """Gradient of ``dropout`` with respect to x (that of residual is dy)."""
    return _dropout(dy, "dy", rate, seed, offset, None, out)


# ---------------------------------------------------------------- gated layer

def _gated_args(x, w_gate, w_up, b_gate, b_up, activation):
    dtype, code, index, stream = _first(x, "x")
    act = ACTIVATIONS.get(activation) if isinstance(activation, str) else None
    if act is None:
        raise ValueError(f"unknown activation {activation!r}; one of {sorted(ACTIVATIONS)}")
    px, rows, width, stride = _rows(x, "x", dtype, index)
    pg, hidden, w_width, g_stride = _rows(w_gate, "w_gate", dtype, index)
    if w_gate.dim() != 2 or w_width != width or hidden == 0:
        raise ValueError(f"w_gate must have shape (hidden, {width}), got {tuple(w_gate.shape)}")
    pu, _, _, u_stride = _rows(w_up, "w_up", dtype, index, w_gate.shape)
    bg = _vector(b_gate, "b_gate", hidden, dtype, index)
    bu = _vector(b_up, "b_up", hidden, dtype, index)
    return (_lib.GatedLayer(code, act, rows, width, hidden, px, stride, pg, g_stride, pu,
                            u_stride, bg, bu), (*x.shape[:-1], hidden), dtype, index, stream)


def _gated_workspace(a, x, backward):
    nbytes = C.c_int64(0)
    _lib.call("mgp_gated_layer_workspace", C.byref(a), backward, C.byref(nbytes))
    return _workspace(x, nbytes.value), nbytes.value


def gated_layer(x, w_gate, w_up, b_gate=None, b_up=None, *, activation="silu", out=None):
    """``act(x w_gate^T + b_gate) * (x w_up^T + b_up)`` in one kernel.

    x [..., width], weights [hidden, width], biases [hidden] or None, all of one
    element type; result [..., hidden].  activation: "silu", "gelu" (with the
    normal distribution's exact integral), "sigmoid" or "relu".  ``out`` shares no
    memory with the inputs."""
    a, shape, dtype, index, stream = _gated_args(x, w_gate, w_up, b_gate, b_up, activation)
    out, ph, h_stride = _result(out, "out", x, shape, dtype, index)
    ws, nbytes = _gated_workspace(a, x, 0)
    _lib.call("mgp_gated_layer_device", C.byref(a), ph, h_stride, _address(ws), nbytes, stream)
    return out


def gated_layer_backward(dh, x, w_gate, w_up, b_gate=None, b_up=None, *, activation="silu",
                         need_dx=True, need_dw=True):
    """Gradients of ``gated_layer`` as ``GatedGradients(dx, dw_gate, dw_up, db_gate, db_up)``.

    The projections are formed again from x: nothing is kept between the
    passes.  In the 16-bit types the gradients of g and u are rounded to the type
    (float16: times a power of two for each row) before the last products; up to 128
    rows they go in two parts.  ``need_dx=False`` (the first layer, whose x is data) and
    ``need_dw=False`` leave those products out."""
    a, shape, dtype, index, stream = _gated_args(x, w_gate, w_up, b_gate, b_up, activation)
    pdh, _, _, dh_stride = _rows(dh, "dh", dtype, index, shape)
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
