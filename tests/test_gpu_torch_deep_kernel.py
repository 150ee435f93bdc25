"""The deep-kernel example: its gradient is the marginal likelihood's, and training
on it fits what a kernel of the inputs does not."""

import importlib.util
from pathlib import Path

import numpy as np
import pytest
import torch

from mojogp_amd._provider import NativeProvider
from oracle import layers as ol

pytestmark = pytest.mark.gpu

PATH = Path(__file__).resolve().parents[1] / "examples" / "deep_kernel.py"


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("deep_kernel", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_gradient_through_the_layers(example):
    """Every weight's gradient of the exact NLL (probes sqrt(n) I: their outer
    products sum to the identity) along random directions, against central
    differences of a float64 NLL over features of the float32 layers."""
    n = 80
    rng = np.random.default_rng(0)
    x = torch.from_numpy(rng.standard_normal((n, 5))).float().cuda()
    y = rng.standard_normal(n).astype(np.float32)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    model = example.Features(5, 24, 3, torch.float32, gen)
    theta, noise = np.array([0.9, 1.1, 1.0, 1.2]), 0.3

    def nll():
        z = model.forward(x, offset=40)[0].double().cpu().numpy()
        K = ol.kernel("rbf", True, z, theta) + noise * np.eye(n)
        return 0.5 * y @ np.linalg.solve(K, y) + 0.5 * np.linalg.slogdet(K)[1]

    z, tape = model.forward(x, offset=40)
    p = NativeProvider("rbf", True, z.cpu().numpy(), theta, noise)
    try:
        probes = np.sqrt(n) * torch.eye(n, device="cuda")
        _, dz, _ = example.likelihood_gradients(p, torch.from_numpy(y).cuda(), probes, tol=1e-6)
    finally:
        p.close()
    step = 2e-3
    for w, g in zip(model.parameters(), model.backward(dz, tape)):
        v = torch.from_numpy(rng.standard_normal(tuple(w.shape))).float().cuda()
        v /= v.norm()
        keep, f = w.clone(), []
        for s in (step, -step):
            w.copy_(keep + s * v)
            f.append(nll())
        w.copy_(keep)
        want = (f[0] - f[1]) / (2 * step)
        # features rounded to 1e-7 of order one move the NLL (gradients of order
        # 10 in 240 coordinates) by 1e-5 over a step of 4e-3; truncation step^2
        got = float((g * v).sum())
        assert abs(got - want) <= 1e-2 * float(g.norm()) + 5e-3


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_training_learns_the_step(example, kind):
    x, y = example.data(2000, seed=3)
    model, theta, history = example.train(x[:1500], y[:1500], kind=kind, report=None)
    assert np.all(np.isfinite(history))
    mean = example.predict(model, theta, x[:1500], y[:1500], x[1500:])
    rmse = float(np.sqrt(np.mean((mean - y[1500:]) ** 2)))
    # a fit that has learnt nothing leaves the labels' spread of one
    assert rmse < 0.7 * float(y[1500:].std())
