"""The layers of a deep kernel: learned features in front of a Gaussian process.

    h = gated_layer(x, w_gate, w_up, b_gate, b_up)      # act(x Wg^T + bg) * (x Wu^T + bu)
    y, saved = layer_norm(h, weight, bias, save=True)
    z = dropout(y, 0.1, seed, offset=step * y.numel())

and their gradients (``gated_layer_backward``, ``layer_norm_backward``,
``dropout_backward``); ``group_norm`` with its activation for features that have
positions, and ``group_norm_backward``; for serving what was trained, layers whose
weights are 8-bit integers (``int8_weights``, ``int8_layer``, ``int8_gated_layer``).  The gradient that enters at the top is
``NativeProvider.input_gradient_device``: that of the marginal likelihood with
respect to the kernel's points.

Arrays are device tensors of the calling program (float32, bfloat16 or
float16, unit stride along the last dimension, leading dimensions that collapse
to one row stride).  Their addresses go to the library's kernels; torch is not
imported here and computes nothing, it provides the arrays, the memory of the
results and the current stream, on which every call runs asynchronously.  The
calls are explicit forward and backward passes and take no part in autograd: an
array that requires a gradient is refused unless torch.no_grad() says that none is
recorded.  A result that the caller gives (``out``) counts as changed in place: a graph of
torch's that saved it refuses its backward pass.
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


def _written(a):
    """To torch's autograd a result that the caller gave has changed in place."""
    if a is not None:
        _torch().autograd.graph.increment_version(a)


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
    _written(out)
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


# ---------------------------------------------------------------- group norm

def _activation(activation):
    if activation is None:
        return -1
    act = ACTIVATIONS.get(activation) if isinstance(activation, str) else None
    if act is None:
        raise ValueError(f"unknown activation {activation!r}; one of {sorted(ACTIVATIONS)} or None")
    return act


def _group_args(x, groups, weight, bias, eps, activation):
    dtype, code, index, stream = _first(x, "x")
    act = _activation(activation)
    if x.dim() < 2:
        raise ValueError(f"x must have shape (samples, ..., channels), got {tuple(x.shape)}")
    px, rows, width, stride = _rows(x, "x", dtype, index)
    samples = x.shape[0]
    positions = 1
    for size in x.shape[1:-1]:
        positions *= size
    if not isinstance(groups, int) or groups < 1 or width % groups:
        raise ValueError(f"groups must divide the {width} channels, got {groups!r}")
    given = weight if weight is not None else bias
    ptype, pcode = dtype, code
    if given is not None and getattr(given, "dtype", None) is not dtype:
        ptype = getattr(given, "dtype", type(given).__name__)
        pcode = _types.get(ptype)
        if pcode != 0:
            raise TypeError(f"weight and bias must have x's element type or be float32, got "
                            f"{ptype}, which does not fit {dtype}")
    pw = _vector(weight, "weight", width, ptype, index)
    pb = _vector(bias, "bias", width, ptype, index)
    return (_lib.GroupNorm(code, pcode, act, eps, samples, positions, width, groups, px, stride,
                           pw, pb), dtype, index, stream)


def _group_workspace(a, x, backward):
    nbytes = C.c_int64(0)
    _lib.call("mgp_group_norm_workspace", C.byref(a), backward, C.byref(nbytes))
    return _workspace(x, nbytes.value), nbytes.value


def group_norm(x, groups, weight=None, bias=None, eps=1e-5, *, activation=None, save=False,
               out=None):
    """Group norm with an activation, channels last: ``act((x - mean) / sqrt(var + eps) *
    weight + bias)``.

    x [samples, ..., channels] (positions between the two, if any); mean and variance
    of each sample are those of all its positions and of ``channels / groups``
    consecutive channels.  weight and bias ([channels], of x's type or float32) may be
    None; activation: None or one of ``gated_layer``'s.  ``out`` may be x, but share no
    memory with it otherwise.  With ``save=True`` returns ``(y, saved)``, ``saved`` being
    what the backward pass takes (mean and reciprocal deviation of every sample's
    groups, float32)."""
    a, dtype, index, stream = _group_args(x, groups, weight, bias, eps, activation)
    y, py, stride = _result(out, "out", x, x.shape, dtype, index)
    stats = x.new_empty((a.samples, groups, 2), dtype=_torch().float32) if save else None
    ws, nbytes = _group_workspace(a, x, 0)
    _lib.call("mgp_group_norm_device", C.byref(a), py, stride, _address(stats), _address(ws),
              nbytes, stream)
    _written(out)
    return (y, stats) if save else y


def group_norm_backward(dy, x, groups, weight, bias, saved, *, activation=None):
    """Gradients ``(dx, dweight, dbias)`` of ``group_norm(x, groups, weight, bias)`` with
    the same activation; None for what is None.  What goes into the activation is
    formed again from x: nothing but ``saved`` is kept between the passes."""
    a, dtype, index, stream = _group_args(x, groups, weight, bias, 0.0, activation)
    pdy, _, _, dy_stride = _rows(dy, "dy", dtype, index, x.shape)
    if getattr(saved, "shape", None) != (a.samples, groups, 2) or _types.get(saved.dtype) != 0 \
            or not saved.is_contiguous() or saved.get_device() != index:
        raise ValueError("saved must be what group_norm(..., save=True) returned for this x")
    dx = x.new_empty(x.shape)
    dweight = None if weight is None else weight.new_empty((a.channels,))
    dbias = None if bias is None else bias.new_empty((a.channels,))
    ws, nbytes = _group_workspace(a, x, 1)
    _lib.call("mgp_group_norm_backward_device", C.byref(a), pdy, dy_stride, saved.data_ptr(),
              dx.data_ptr(), a.channels, _address(dweight), _address(dbias), _address(ws), nbytes,
              stream)
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
    _written(out)
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
    h, ph, h_stride = _result(out, "out", x, shape, dtype, index)
    ws, nbytes = _gated_workspace(a, x, 0)
    _lib.call("mgp_gated_layer_device", C.byref(a), ph, h_stride, _address(ws), nbytes, stream)
    _written(out)
    return h


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


# ---------------------------------------------------------------- layers in 8-bit integers

class Int8Weights(NamedTuple):
    """What int8_weights returns: codes (int8, [rows, width rounded up to 16], zeros
    behind width), a float32 scale for each row, and the width."""
    codes: object
    scale: object
    width: int


def int8_weights(w):
    """Weights [hidden, width] as 8-bit integers with a scale for each row, for
    ``int8_layer`` and ``int8_gated_layer``: half the bytes of 16-bit ones.

    The codes are -127 .. 127, the row times 127 over its largest value, rounded to
    even.  A row that is not finite gets the scale NaN.  At most 131072 columns."""
    dtype, code, index, stream = _first(w, "w")
    pw, rows, width, stride = _rows(w, "w", dtype, index)
    if w.dim() != 2:
        raise ValueError(f"w must have shape (hidden, width), got {tuple(w.shape)}")
    torch = _torch()
    padded = -(-width // 16) * 16
    codes = w.new_empty((rows, padded), dtype=torch.int8)
    scale = w.new_empty((rows,), dtype=torch.float32)
    _lib.call("mgp_int8_quantize_device", code, pw, stride, rows, width, codes.data_ptr(), padded,
              scale.data_ptr(), stream)
    return Int8Weights(codes, scale, width)


def _int8_side(w, name, width, index, hidden=None):
    """(codes' address, scales' address, rows, row stride)"""
    if not isinstance(w, Int8Weights):
        raise TypeError(f"{name} must be what int8_weights returned, got {type(w).__name__}")
    codes, scale, columns = w
    _check(codes, f"{name}.codes", _torch().int8, index)
    shape = codes.shape
    rows = shape[0] if len(shape) == 2 else 0
    if columns != width or shape != (rows, -(-width // 16) * 16) or not codes.is_contiguous():
        raise ValueError(f"{name} must be weights of {width} columns, got {columns} in codes of "
                         f"shape {tuple(shape)}")
    if rows == 0 or (hidden is not None and rows != hidden):
        raise ValueError(f"{name} must have {hidden or 'at least one'} rows, got {rows}")
    return codes.data_ptr(), _vector(scale, f"{name}.scale", rows, _torch().float32, index), rows


def _int8(x, gate, up, b_gate, b_up, act, names, out):
    dtype, code, index, stream = _first(x, "x")
    px, rows, width, stride = _rows(x, "x", dtype, index)
    wg, sg, hidden = _int8_side(gate, names[0], width, index)
    wu = su = None
    if up is not None:
        wu, su, _ = _int8_side(up, names[1], width, index, hidden)
    bg = _vector(b_gate, names[2], hidden, dtype, index)
    bu = _vector(b_up, names[3], hidden, dtype, index)
    a = _lib.Int8Layer(code, act, rows, width, hidden, px, stride, wg, wu, gate.codes.shape[1], sg,
                       su, bg, bu)
    y, py, y_stride = _result(out, "out", x, (*x.shape[:-1], hidden), dtype, index)
    nbytes = C.c_int64(0)
    _lib.call("mgp_int8_layer_workspace", C.byref(a), C.byref(nbytes))
    ws = _workspace(x, nbytes.value)
    _lib.call("mgp_int8_layer_device", C.byref(a), py, y_stride, _address(ws), nbytes.value, stream)
    _written(out)
    return y


def int8_layer(x, weights, bias=None, *, activation=None, out=None):
    """``act(x w^T + bias)`` with weights from ``int8_weights`` and each row of x rounded
    to 8 bits in the same way, the sums being exact.

    x [..., width] and bias [hidden] (or None) of one element type, which the result
    [..., hidden] has too; activation: None or one of ``gated_layer``'s.  Rows that
    are not finite give NaN.  ``out`` shares no memory with the inputs."""
    return _int8(x, weights, None, bias, None, _activation(activation),
                 ("weights", "", "bias", ""), out)


def int8_gated_layer(x, w_gate, w_up, b_gate=None, b_up=None, *, activation="silu", out=None):
    """``gated_layer`` with weights from ``int8_weights``, and x as in ``int8_layer``."""
    act = _activation(activation)
    if act < 0:
        raise ValueError(f"unknown activation None; one of {sorted(ACTIVATIONS)}")
    return _int8(x, w_gate, w_up, b_gate, b_up, act, ("w_gate", "w_up", "b_gate", "b_up"), out)
