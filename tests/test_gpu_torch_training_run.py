"""Layers with positions, trained by AdamW and served in 8-bit integers: the calls
one after another as a program makes them, each held to its float64 formula on what
the call before it left, and the chain's gradient to differences."""

import importlib.util
from pathlib import Path

import numpy as np
import pytest
import torch

from mojogp_amd import features, optim
from oracle import layers as ol
from oracle import optim as oo

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
UNIT = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
F32 = 1e-5  # fp32 sums of up to 2000 terms and the activations, as in the layers' own tests
N, L, WIDTH, HIDDEN, GROUPS = 30, 7, 24, 40, 5


def _host(t):
    return t.double().cpu().numpy()


def _near(got, want, tol):
    assert np.linalg.norm(_host(got) - want) <= tol * np.linalg.norm(want)


class Model:
    """x -> gated layer -> group norm with an activation -> gated layer."""

    def __init__(self, rng, dtype):
        def t(*shape, scale=1.0, shift=0.0):
            return torch.from_numpy(scale * rng.normal(size=shape) + shift).to("cuda", dtype)

        self.first = [t(HIDDEN, WIDTH, scale=WIDTH ** -0.5), t(HIDDEN, WIDTH, scale=WIDTH ** -0.5),
                      t(HIDDEN, scale=0.1), t(HIDDEN, scale=0.1)]
        self.norm = [t(HIDDEN, scale=0.1, shift=1.0), t(HIDDEN, scale=0.1)]
        self.last = [t(3, HIDDEN, scale=HIDDEN ** -0.5), t(3, HIDDEN, scale=HIDDEN ** -0.5),
                     t(3, scale=0.1), t(3, scale=0.1)]

    def parameters(self):
        return [*self.first, *self.norm, *self.last]

    def forward(self, x):
        h = features.gated_layer(x, *self.first)
        y, saved = features.group_norm(h, GROUPS, *self.norm, activation="silu", save=True)
        return features.gated_layer(y, *self.last, activation="gelu"), (x, h, y, saved)

    def backward(self, dz, tape):
        x, h, y, saved = tape
        last = features.gated_layer_backward(dz, y, *self.last, activation="gelu")
        dh, *norm = features.group_norm_backward(last.dx, h, GROUPS, *self.norm, saved,
                                                 activation="silu")
        first = features.gated_layer_backward(dh, x, *self.first, need_dx=False)
        return [*first[1:], *norm, *last[1:]]

    def serve(self):
        first = [*map(features.int8_weights, self.first[:2]), *self.first[2:]]
        last = [*map(features.int8_weights, self.last[:2]), *self.last[2:]]

        def z(x):
            h = features.int8_gated_layer(x, *first)
            y = features.group_norm(h, GROUPS, *self.norm, activation="silu")
            return features.int8_gated_layer(y, *last, activation="gelu"), h, y

        return z


def _x(rng, dtype):
    return torch.from_numpy(rng.normal(size=(N, L, WIDTH))).to("cuda", dtype)


def test_gradient_against_differences():
    """Of the float32 chain along random directions: values of size 60 (N L 3 terms of
    order one, dz of order one) rounded to 1e-6 over a step of 4e-3, truncation step^2."""
    rng = np.random.default_rng(0)
    model, x = Model(rng, torch.float32), _x(rng, torch.float32)
    dz = torch.from_numpy(rng.normal(size=(N, L, 3))).float().cuda()
    z, tape = model.forward(x)
    grads, step = model.backward(dz, tape), 2e-3
    for p, g in zip(model.parameters(), grads):
        assert p.shape == g.shape
        v = torch.from_numpy(rng.normal(size=tuple(p.shape))).float().cuda()
        v /= v.norm()
        keep, f = p.clone(), []
        for s in (step, -step):
            p.copy_(keep + s * v)
            f.append(float((model.forward(x)[0].double() * dz.double()).sum()))
        p.copy_(keep)
        want = (f[0] - f[1]) / (2 * step)
        assert abs(float((g.double() * v.double()).sum()) - want) <= 2e-2 + 2e-3 * float(g.norm())


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("kind", sorted(TYPES))
def test_steps_and_serving(kind, bits):
    rng = np.random.default_rng(bits)
    dtype, u = TYPES[kind], UNIT[kind]
    model, x = Model(rng, dtype), _x(rng, dtype)
    master = kind != "f32"
    opt = optim.AdamW(model.parameters(), bits=bits, master=master, betas=(0.9, 0.99), seed=4)
    for step in (1, 2, 3):
        z, tape = model.forward(x)
        x_, h, y, saved = tape
        dz = (z.float() * 0.1).to(dtype)
        grads = model.backward(dz, tape)
        # each call against its formula on the arrays before it
        norm = [_host(p) for p in model.norm]
        _near(y, ol.group_norm(_host(h), GROUPS, *norm, act="silu"), u + F32)
        flat = [_host(t).reshape(N * L, -1) for t in (dz, y)]
        dy = ol.gated_layer_backward(flat[0], flat[1], *map(_host, model.last), act="gelu")[0]
        # (dy carries the rounding of dg and du and its own, 3 u; the channels' sums of up
        # to N L of them cancel less than tenfold here)
        ref = ol.group_norm_backward(dy.reshape(N, L, HIDDEN), _host(h), GROUPS, *norm, act="silu")
        for got, want in zip(grads[4:6], ref[1:]):
            _near(got, want, 30 * u + 10 * F32)
        before = [_host(t) for t in opt.split(opt.master)] if master else \
            [_host(p) for p in model.parameters()]
        means = [[_host(t).ravel() for t in opt.split(v)] for v in
                 (opt.values()["exp_avg"], opt.values()["exp_avg_sq"])]
        total, factor = oo.clip([_host(g) for g in grads], 0.5)
        got = opt.step(grads, 0.01, step, max_norm=0.5)
        assert abs(float(got) - total) <= 2e-7 * total
        after = opt.split(opt.master) if master else model.parameters()
        for p, old, g, m, v in zip(after, before, grads, *means):
            m, v = oo.moments(m, v, _host(g).ravel() * factor, (0.9, 0.99))
            want = oo.update(old.ravel(), m, v, 0.01, step, (0.9, 0.99), 1e-8, 0.0)
            # fp32 operations of a step of 0.01 or so beside two roundings of the value
            assert np.abs(_host(p).ravel() - want).max() <= 1e-6 * np.abs(want).max() + 1e-6
    served, h, y = model.serve()(x)
    first, last = (list(map(_host, t)) for t in (model.first, model.last))
    wg, wu, bg, bu = first
    want, _ = ol.int8_layer(_host(x).reshape(N * L, -1), wg, bg, wu, bu, "silu")
    _near(h.view(N * L, -1), want, u + F32)
    wg, wu, bg, bu = last
    want, _ = ol.int8_layer(_host(y).reshape(N * L, -1), wg, bg, wu, bu, "gelu")
    _near(served.view(N * L, -1), want, u + F32)


def test_a_recorded_step():
    """Forward, backward and the optimiser's step in one graph, replayed with eager
    work between, give what single calls give."""
    rng = np.random.default_rng(3)
    one, two = Model(np.random.default_rng(1), torch.bfloat16), Model(np.random.default_rng(1),
                                                                      torch.bfloat16)
    x = _x(rng, torch.bfloat16)
    opts = [optim.AdamW(m.parameters(), bits=8, master=True, seed=2) for m in (one, two)]
    number = torch.ones((), device="cuda", dtype=torch.int64)
    rate = torch.full((), 0.01, device="cuda")

    def step(model, opt, number, rate):
        z, tape = model.forward(x)
        opt.step(model.backward(z, tape), rate, number, max_norm=1.0)
        return z

    start = [p.clone() for p in one.parameters()], {k: t.clone() for k, t in opts[0].state().items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(one, opts[0], number, rate)
    torch.cuda.current_stream().wait_stream(side)
    for p, q in zip(one.parameters(), start[0]):
        p.copy_(q)
    opts[0].load(start[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        z = step(one, opts[0], number, rate)
    for t in range(1, 5):
        number.fill_(t)
        x.copy_(_x(rng, torch.bfloat16))
        graph.replay()
        assert torch.equal(z, step(two, opts[1], t, float(rate)))
        for p, q in zip(one.parameters(), two.parameters()):
            assert torch.equal(p, q)


@pytest.mark.parametrize("kind, bits", [("f32", 8), ("bf16", 8), ("f16", 32)])
def test_the_deep_kernel_example_runs(kind, bits):
    """With 8-bit states, and served in 8-bit integers."""
    path = Path(__file__).resolve().parents[1] / "examples" / "deep_kernel.py"
    spec = importlib.util.spec_from_file_location("deep_kernel", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    x, y = example.data(600, seed=1)
    model, theta, history = example.train(x[:500], y[:500], kind=kind, bits=bits, steps=3,
                                          report=None)
    assert len(history) == 3 and np.isfinite(history).all()
    for int8 in (False, True):
        assert np.isfinite(example.predict(model, theta, x[:500], y[:500], x[500:], int8)).all()
