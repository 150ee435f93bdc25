"""The step that trains the layers of mojogp_amd.features: AdamW over all their
parameters at once.

    opt = AdamW(layers.parameters(), bits=8, weight_decay=0.01)
    for t in range(1, steps + 1):
        grads = ...                      # by the layers' backward passes
        norm = opt.step(grads, 1e-3, t, max_norm=1.0)

Parameters and gradients are device tensors of the calling program, as in
mojogp_amd.features; the states belong to the optimiser.  A step is one launch for
hundreds of tensors (two more where the norm of all gradients is formed), runs
asynchronously on the current stream and can be recorded into a graph.
"""

from __future__ import annotations

import array
import ctypes as C
import math
import numbers
import operator

import numpy as np

from . import _lib
from .features import _no_graph, _stream, _torch, _types

_FLOAT_MOST = float(np.finfo(np.float32).max)
_required, _shape_of, _dtype_of = map(operator.attrgetter, ("requires_grad", "shape", "dtype"))


class AdamW:
    """AdamW (decoupled weight decay) with states in 32 or in 8 bits.

    params: contiguous float32, bfloat16 or float16 device tensors, all of one
    type, which share no memory; they are changed in place, always at the addresses
    that they have here.  ``master=True`` (16-bit types) keeps float32 copies, which
    the steps change and the parameters are rounded from: without them a step below
    the parameter's last bit is lost.  weight_decay: one number, or one for each
    parameter.

    ``bits=8`` holds the running means as 8-bit floats with a float32 scale for each
    256 values of a parameter (2.03 bytes a value instead of 8), rounded up or down by
    draws that are functions of ``seed``, the step and the value's place alone.  The
    update itself is formed before the rounding.  A gradient that is not finite makes
    NaN of the states of its scale's 256 values, and one whose square passes float32 (by
    about a thousandfold at the default betas) of their second means, where ``step``
    forms no norm that catches it.

    exp_avg, exp_avg_sq (float32, or codes with exp_avg_scale and exp_avg_sq_scale) and
    master are flat arrays in which each parameter's values start at the next multiple
    of 256; ``split`` makes views of them in the parameters' shapes."""

    def __init__(self, params, *, bits=32, master=False, betas=(0.9, 0.999), eps=1e-8,
                 weight_decay=0.0, seed=0):
        torch = _torch()
        self.params = list(params)
        if not self.params:
            raise ValueError("params must hold at least one tensor")
        first = self.params[0]
        self._dtype = getattr(first, "dtype", None)
        code = _types.get(self._dtype)
        if code is None:
            raise TypeError("params must be float32, bfloat16 or float16 device tensors, got "
                            f"{self._dtype or type(first).__name__}")
        self._index = first.get_device()
        if self._index < 0:
            raise ValueError(f"params must be device tensors, got one on {first.device}")
        for i, p in enumerate(self.params):
            self._check(p, f"params[{i}]", self._dtype)
        self._shapes = [p.shape for p in self.params]
        self._addresses = [p.data_ptr() for p in self.params]
        decays = [weight_decay] * len(self.params) if isinstance(weight_decay, numbers.Real) \
            else list(weight_decay)
        if len(decays) != len(self.params):
            raise ValueError(f"weight_decay must be a number or {len(self.params)} of them, got "
                             f"{len(decays)}")
        if isinstance(seed, bool) or not isinstance(seed, numbers.Integral) \
                or not 0 <= seed < 1 << 64:
            raise ValueError("seed must be an integer in [0, 2^64)")
        tensors = (_lib.AdamWTensor * len(self.params))(*[
            (a, p.numel(), d) for a, p, d in zip(self._addresses, self.params, decays)])
        a = _lib.AdamW(type=code, bits=bits, master_copies=bool(master), count=len(self.params),
                       tensors=tensors, beta1=betas[0], beta2=betas[1], eps=eps, seed=int(seed))
        values, nbytes = C.c_int64(0), C.c_int64(0)
        _lib.call("mgp_adamw_layout", C.byref(a), C.byref(values), C.byref(nbytes))
        self.bits, n = bits, values.value

        def zeros(count, dtype):
            return first.new_zeros(count, dtype=dtype, requires_grad=False)

        state = torch.uint8 if bits == 8 else torch.float32
        self.exp_avg, self.exp_avg_sq = zeros(n, state), zeros(n, state)
        self.exp_avg_scale = self.exp_avg_sq_scale = self.master = None
        if bits == 8:
            self.exp_avg_scale = zeros(n // 256, torch.float32)
            self.exp_avg_sq_scale = zeros(n // 256, torch.float32)
        if master:
            self.master = zeros(n, torch.float32)
            for view, p in zip(self.split(self.master), self.params):
                view.copy_(p.detach())
        host = np.zeros(nbytes.value, dtype=np.uint8)
        self._table = zeros(nbytes.value, torch.uint8)
        for name in ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale", "master"):
            t = getattr(self, name)
            setattr(a, name, None if t is None else t.data_ptr())
        a.table = self._table.data_ptr()
        plan = C.c_void_p()
        _lib.call("mgp_adamw_create", C.byref(a), host.ctypes.data, host.size, C.byref(plan))
        self._plan = plan.value
        self._table.copy_(torch.from_numpy(host))
        s = _lib.AdamWStep(grads=(C.c_void_p * len(self.params))(), grad_type=code, form_norm=1,
                           grad_scale=1.0, max_norm=1.0, step=1)
        _lib.call("mgp_adamw_workspace", self._plan, C.byref(s), C.byref(nbytes))
        self._workspace = nbytes.value

    def _check(self, t, name, dtype):
        if getattr(t, "dtype", None) is not dtype:
            raise TypeError(f"{name} must be a {dtype} tensor, got "
                            f"{getattr(t, 'dtype', type(t).__name__)}")
        if t.requires_grad:
            _no_graph(name)
        if t.get_device() != self._index:
            raise ValueError(f"{name} must be on device {self._index}, got {t.device}")
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")

    def split(self, flat):
        """Views of a flat state array in the parameters' shapes."""
        views, at = [], 0
        for p in self.params:
            views.append(flat[at:at + p.numel()].view(p.shape))
            at += -(-p.numel() // 256) * 256
        return views

    def _addresses_of(self, grads, dtype):
        """Gradients' addresses, each checked."""
        tensor = _torch().Tensor
        if set(map(type, grads)) == {tensor} and set(map(tensor.get_device, grads)) == {self._index} \
                and all(map(tensor.is_contiguous, grads)) \
                and set(map(_dtype_of, grads)) == {dtype} and not any(map(_required, grads)) \
                and list(map(_shape_of, grads)) == self._shapes:
            return list(map(tensor.data_ptr, grads))
        out, index = [], self._index  # one by one: None among them, or one to be named
        for i, (g, shape) in enumerate(zip(grads, self._shapes)):
            if g is None:
                out.append(0)
                continue
            if getattr(g, "dtype", None) is not dtype or g.shape != shape or g.requires_grad \
                    or not g.is_contiguous() or g.get_device() != index:
                self._check(g, f"grads[{i}]", dtype)
                if g.shape != shape:
                    raise ValueError(f"grads[{i}] must have shape {tuple(shape)}, got "
                                     f"{tuple(g.shape)}")
            out.append(g.data_ptr())
        return out

    def _scalar(self, t, name, dtype):
        """Address of a device scalar."""
        self._check(t, name, dtype)
        if t.numel() != 1:
            raise ValueError(f"{name} must have one element, got {t.numel()}")
        return t.data_ptr()

    def step(self, grads, rate, step, *, max_norm=None, norm=False, grad_scale=1.0):
        """One step: ``grads`` hold a gradient for each parameter (of the parameters'
        type, or all float32), None for those that are left as they are.

        rate and step (1 at the first step) are numbers, or device tensors of one
        element (float32, int64), which a recorded graph reads at every replay (the
        optimizer has to live as long as the graph); where such a step is below 1, or such a
        rate negative or not finite, everything is left as it is.
        The gradients are multiplied by ``grad_scale`` and, where ``max_norm`` is
        given, by max_norm over their common norm if that is larger.  With max_norm or
        ``norm=True`` the norm comes back (float32, on the device), and a norm that is
        not finite leaves everything unchanged.

        To torch's autograd a step changes its parameters in place: a graph that saved one
        refuses its backward pass afterwards.  (Replays of a recorded graph go unnoticed.)"""
        torch = _torch()
        if self._plan is None:
            raise ValueError("the optimizer is closed")
        current = torch.cuda.current_device()
        if current != self._index:
            raise ValueError(f"the parameters are on device {self._index}, the current device "
                             f"is {current}")
        if torch.is_grad_enabled():
            if any(map(_required, self.params)):
                _no_graph(f"params[{list(map(_required, self.params)).index(True)}]")
        if list(map(torch.Tensor.data_ptr, self.params)) != self._addresses:
            raise ValueError("the parameters' memory is no longer where it was when the optimizer "
                             "was made")
        grads = list(grads)
        if len(grads) != len(self.params):
            raise ValueError(f"{len(self.params)} gradients are needed, got {len(grads)}")
        dtype = next((getattr(g, "dtype", None) for g in grads if g is not None), self._dtype)
        if dtype is not self._dtype and dtype is not torch.float32:
            raise TypeError(f"gradients must be of the parameters' type ({self._dtype}) or "
                            f"float32, got {dtype}")
        pointers = array.array("Q", self._addresses_of(grads, dtype))
        s = _lib.AdamWStep(grads=C.cast(pointers.buffer_info()[0], _lib.c_void_pp),
                           grad_type=_types[dtype], grad_scale=grad_scale, max_norm=math.inf)
        if isinstance(step, numbers.Integral) and not isinstance(step, bool):
            if not 1 <= step < 1 << 53:
                raise ValueError(f"step must be at least 1, got {step}")
            s.step = int(step)
        else:
            s.step_device = self._scalar(step, "step", torch.int64)
        if isinstance(rate, numbers.Real):
            if not 0 <= rate <= _FLOAT_MOST:
                raise ValueError(f"the rate must be finite and >= 0, got {rate}")
            s.rate = rate
        else:
            s.rate_device = self._scalar(rate, "rate", torch.float32)
        result = ws = None
        if norm or max_norm is not None:
            s.form_norm = 1
            if max_norm is not None:
                s.max_norm = max_norm
            result = self.exp_avg.new_empty((), dtype=torch.float32)
            s.norm = result.data_ptr()
        nbytes = 0
        if result is not None or s.step_device or s.rate_device:
            nbytes = self._workspace
            ws = self.exp_avg.new_empty(nbytes, dtype=torch.uint8)
        _lib.call("mgp_adamw_step_device", self._plan, C.byref(s),
                  None if ws is None else ws.data_ptr(), nbytes, _stream(torch, current))
        changed = self.params if all(pointers) else [p for p, at in zip(self.params, pointers) if at]
        torch.autograd.graph.increment_version(changed)
        return result

    def values(self):
        """What the states stand for, as flat float32 arrays: ``exp_avg``,
        ``exp_avg_sq`` (new arrays if held in 8 bits, the states themselves otherwise)
        and, if there is one, ``master``."""
        torch = _torch()
        if self._plan is None:
            raise ValueError("the optimizer is closed")
        m, v = self.exp_avg, self.exp_avg_sq
        if self.bits == 8:
            current = torch.cuda.current_device()
            if current != self._index:
                raise ValueError(f"the states are on device {self._index}, the current device is "
                                 f"{current}")
            m, v = (t.new_empty(t.shape, dtype=torch.float32) for t in (m, v))
            _lib.call("mgp_adamw_values_device", self._plan, m.data_ptr(), v.data_ptr(),
                      _stream(torch, current))
        out = {"exp_avg": m, "exp_avg_sq": v}
        if self.master is not None:
            out["master"] = self.master
        return out

    def state(self):
        """The states themselves, by name: what ``load`` takes."""
        names = ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale", "master")
        return {n: getattr(self, n) for n in names if getattr(self, n) is not None}

    def load(self, state):
        """Copies states of the same layout (``state`` of an optimiser of the same
        parameters) into this one's."""
        mine = self.state()
        if set(state) != set(mine):
            raise ValueError(f"states {sorted(mine)} are needed, got {sorted(state)}")
        for name, t in mine.items():
            if state[name].shape != t.shape or state[name].dtype is not t.dtype:
                raise ValueError(f"{name} must be {t.dtype} of shape {tuple(t.shape)}, got "
                                 f"{state[name].dtype} of {tuple(state[name].shape)}")
        for name, t in mine.items():
            t.copy_(state[name])

    def close(self):
        """Ends the plan; the parameters and states stay what they are."""
        plan, self._plan = getattr(self, "_plan", None), None
        if plan is not None:
            _lib.call("mgp_adamw_destroy", plan)

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
