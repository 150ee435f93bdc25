"""The AdamW step's C entry where Python's optim.AdamW does not reach: steps and rates
on the device without a norm, whatever stands in the fields of the norm."""

import ctypes as C

import pytest
import torch

from mojogp_amd import _lib, optim

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("max_norm", [-1.0, 0.0, float("nan"), 1e-3])
@pytest.mark.parametrize("device", ["step", "rate", "both"])
def test_without_a_norm_its_fields_are_not_used(bits, max_norm, device):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(3)
    start = torch.randn(700, device="cuda", generator=gen)
    grad = torch.randn(700, device="cuda", generator=gen)
    params = [start.clone(), start.clone()]
    want, got = (optim.AdamW([p], bits=bits, seed=5) for p in params)
    want.step([grad], 0.125, 3, grad_scale=0.5)
    step = torch.full((), 3, device="cuda", dtype=torch.int64)
    rate = torch.full((), 0.125, device="cuda")
    norm = torch.full((), 7.0, device="cuda")
    s = _lib.AdamWStep(grads=(C.c_void_p * 1)(grad.data_ptr()), grad_type=0, form_norm=0,
                       grad_scale=0.5, max_norm=max_norm, norm=norm.data_ptr(), step=3, rate=0.125)
    if device != "rate":
        s.step_device = step.data_ptr()
    if device != "step":
        s.rate_device = rate.data_ptr()
    nbytes = C.c_int64(0)
    _lib.call("mgp_adamw_workspace", got._plan, C.byref(s), C.byref(nbytes))
    ws = torch.empty(nbytes.value, device="cuda", dtype=torch.uint8)
    _lib.call("mgp_adamw_step_device", got._plan, C.byref(s), ws.data_ptr(), nbytes.value,
              torch.cuda.current_stream().cuda_stream)
    assert torch.equal(params[1], params[0]) and float(norm) == 7.0
    for k, t in want.state().items():
        assert torch.equal(got.state()[k], t)


@pytest.mark.parametrize("steps_on", ["numbers", "device"])
def test_autograd_sees_that_parameters_change(steps_on):
    """A graph of torch's that saved a parameter refuses its backward pass after a step;
    parameters without a gradient are not changed."""
    w = torch.ones(5, device="cuda", requires_grad=True)
    other = torch.ones(5, device="cuda", requires_grad=True)
    with torch.no_grad():
        opt = optim.AdamW([w, other])
    loss, kept = (w * w).sum(), (other * other).sum()
    versions = w._version, other._version
    rate, step = 0.1, 1
    if steps_on == "device":
        rate = torch.full((), 0.1, device="cuda")
        step = torch.ones((), device="cuda", dtype=torch.int64)
    with torch.no_grad():
        opt.step([torch.ones(5, device="cuda"), None], rate, step)
    assert w._version > versions[0] and other._version == versions[1]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    kept.backward()
    assert torch.equal(other.grad, torch.full((5,), 2.0, device="cuda"))
    with torch.inference_mode():  # tensors without versions
        p = torch.ones(5, device="cuda")
        optim.AdamW([p]).step([torch.ones(5, device="cuda")], 0.1, 1)
    assert not torch.equal(p, torch.ones(5, device="cuda"))
