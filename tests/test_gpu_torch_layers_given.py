"""Results in arrays that the caller gives: to torch's autograd they change in place."""

import numpy as np
import pytest
import torch

from mojogp_amd import _lib, features
from mojogp_amd._provider import NativeProvider

pytestmark = pytest.mark.gpu

N, WIDTH = 12, 16


def _input_gradient(x, out):
    rng = np.random.default_rng(0)
    provider = NativeProvider("rbf", True, rng.normal(size=(N, WIDTH)).astype(np.float32),
                              np.ones(WIDTH + 1), 0.1)
    try:
        provider.input_gradient_device(torch.ones(2, N, device="cuda"),
                                       torch.ones(2, N, device="cuda"), out=out)
        torch.cuda.synchronize()
    finally:
        provider.close()


def _weights():
    return torch.ones(WIDTH, WIDTH, device="cuda")


CALLS = {
    "layer norm": lambda x, out: features.layer_norm(x, out=out),
    "group norm": lambda x, out: features.group_norm(x, 2, out=out),
    "dropout": lambda x, out: features.dropout(x, 0.5, 1, out=out),
    "gated layer": lambda x, out: features.gated_layer(x, _weights(), _weights(), out=out),
    "8-bit layer": lambda x, out: features.int8_layer(x, features.int8_weights(_weights()), out=out),
    "input gradient": _input_gradient,
}


@pytest.mark.parametrize("name", sorted(CALLS))
def test_a_graph_that_saved_the_result_refuses_its_backward_pass(name):
    x = torch.randn(N, WIDTH, device="cuda")
    out = torch.randn(N, WIDTH, device="cuda")
    w = torch.ones(N, WIDTH, device="cuda", requires_grad=True)
    loss, other = (w * out).sum(), (w * x).sum()
    CALLS[name](x, out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    other.backward()  # what is only read counts as it was
    assert torch.equal(w.grad, x)


def test_a_refused_call_changes_nothing():
    x = torch.randn(N, WIDTH, device="cuda")
    w = torch.ones(N, WIDTH, device="cuda", requires_grad=True)
    loss = (w * x).sum()
    with pytest.raises(_lib.NativeCallError):
        features.group_norm(x, 2, eps=-1.0, out=x)
    loss.backward()
    assert torch.equal(w.grad, x)
