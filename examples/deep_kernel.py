"""A deep kernel: gated layers, layer norms and dropout in front of a Gaussian process.

    python -m examples.deep_kernel [--points 4000] [--steps 80] [--type bf16] [--bits 8] [--int8]

The features z = f(x), normalised so that they cannot run away from each other,
are the points of an RBF kernel; layers, kernel parameters and noise are trained
on the GP's marginal likelihood:

    NLL = 1/2 y^T K^-1 y + 1/2 log|K|,   K = K(z, z) + noise I

With alpha = K^-1 y, probes Z (Z Z^T / T = I on average) and U = K^-1 Z its
gradient with respect to the points is the input gradient of K for the weight
columns [-alpha / 2 | U / (2 T)] and [alpha | Z]; it goes back through the
layers by their own backward passes, and one AdamW step over all of them, with float32
copies of 16-bit weights and states in 32 or 8 bits, follows.  The trained layers
serve test points in their own type or in 8-bit integers.  torch holds the arrays and
does the vector work of the conjugate gradients.
"""

import argparse
import ctypes as C

import numpy as np
import torch

from mojogp_amd import _lib, features, optim
from mojogp_amd._provider import NativeProvider

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
RATE, SEED = 0.1, 20  # dropout
EPS = 1e-2              # of the last norm: features of no spread stay near zero


class Features:
    """x -> gated -> (norm -> gated -> dropout, residual) -> norm -> gated -> norm = z."""

    def __init__(self, inputs, width, outputs, dtype, generator):
        def weight(rows, cols):
            w = torch.randn(rows, cols, generator=generator, device="cuda") / cols ** 0.5
            return w.to(dtype)

        def bias(rows):
            return torch.zeros(rows, device="cuda", dtype=dtype)

        def norm():
            return [torch.ones(width, device="cuda", dtype=dtype), bias(width)]

        self.first = [weight(width, inputs), weight(width, inputs), bias(width), bias(width)]
        self.norm1, self.norm2 = norm(), norm()
        self.second = [weight(width, width), weight(width, width), bias(width), bias(width)]
        self.last = [weight(outputs, width), weight(outputs, width), bias(outputs), bias(outputs)]

    def parameters(self):
        return [*self.first, *self.norm1, *self.second, *self.norm2, *self.last]

    def forward(self, x, offset=0, rate=None):
        """(z, what backward needs); offset: the first dropout draw of the step."""
        rate = RATE if rate is None else rate
        h0 = features.gated_layer(x, *self.first)
        y0, s0 = features.layer_norm(h0, *self.norm1, save=True)
        g = features.gated_layer(y0, *self.second)
        h1 = features.dropout(g, rate, SEED, offset=offset, residual=h0)
        y1, s1 = features.layer_norm(h1, *self.norm2, save=True)
        f = features.gated_layer(y1, *self.last, activation="gelu")
        z, s2 = features.layer_norm(f, eps=EPS, save=True)
        return z, (x, h0, y0, s0, h1, y1, s1, f, s2, offset, rate)

    def int8(self):
        """z of x with every layer's weights in 8-bit integers: a function, for serving."""
        def weights(layer):
            return [*map(features.int8_weights, layer[:2]), *layer[2:]]

        first, second, last = map(weights, (self.first, self.second, self.last))

        def serve(x):
            h0 = features.int8_gated_layer(x, *first)
            h1 = features.int8_gated_layer(features.layer_norm(h0, *self.norm1), *second) + h0
            f = features.int8_gated_layer(features.layer_norm(h1, *self.norm2), *last,
                                          activation="gelu")
            return features.layer_norm(f, eps=EPS)

        return serve

    def backward(self, dz, tape):
        """Gradients in the order of parameters()."""
        x, h0, y0, s0, h1, y1, s1, f, s2, offset, rate = tape
        df, _, _ = features.layer_norm_backward(dz, f, None, s2, bias=False)
        last = features.gated_layer_backward(df, y1, *self.last, activation="gelu")
        dh1, *norm2 = features.layer_norm_backward(last.dx, h1, self.norm2[0], s1)
        dg = features.dropout_backward(dh1, rate, SEED, offset=offset)
        second = features.gated_layer_backward(dg, y0, *self.second)
        dh0, *norm1 = features.layer_norm_backward(second.dx, h0, self.norm1[0], s0)
        first = features.gated_layer_backward(dh0 + dh1, x, *self.first, need_dx=False)
        return [*first[1:], *norm1, *second[1:], *norm2, *last[1:]]


def _product(provider, v, out):
    """(K + noise I) v of device columns [t, n]."""
    torch.cuda.current_stream().synchronize()  # the provider has a stream of its own
    _lib.call("mgp_forward_matvec_device", provider.handle,
              C.cast(v.data_ptr(), C.POINTER(C.c_float)), v.shape[0],
              C.cast(out.data_ptr(), C.POINTER(C.c_float)))
    return out


def solve(provider, b, tol=1e-3, iterations=500):
    """(K + noise I)^-1 b by conjugate gradients, a column each row of b."""
    x, r, q = torch.zeros_like(b), b.clone(), b.clone()
    kq = torch.empty_like(b)
    rr = (r * r).sum(dim=1, keepdim=True)
    stop = tol * tol * rr
    for _ in range(iterations):
        if bool((rr <= stop).all()):
            break
        _product(provider, q, kq)
        step = rr / (q * kq).sum(dim=1, keepdim=True).clamp_min(1e-30)
        x += step * q
        r -= step * kq
        new = (r * r).sum(dim=1, keepdim=True)
        q = r + (new / rr.clamp_min(1e-30)) * q
        rr = new
    return x


def likelihood_gradients(provider, y, probes, tol=1e-3):
    """(y^T K^-1 y, d NLL / d points, d NLL / d [kernel parameters, noise]) of the
    provider's kernel; y [n], probes [T, n] (device)."""
    t = probes.shape[0]
    u = solve(provider, torch.cat([y[None], probes]), tol)
    left = torch.cat([-0.5 * u[:1], u[1:] / (2.0 * t)])
    right = torch.cat([u[:1], probes])
    points = provider.input_gradient_device(left, right)
    kernel = provider.gradient_trace(left.cpu().numpy(), right.cpu().numpy())
    return float((y * u[0]).sum()), points, np.append(kernel, float((left * right).sum()))


class Adam:
    """Of the kernel's parameters, which are on the host."""

    def __init__(self, rate):
        self.rate, self.step, self.state = rate, 0, {}

    def update(self, params, grads):
        """New values of arrays."""
        self.step += 1
        out = []
        for i, (p, g) in enumerate(zip(params, grads)):
            m, v = self.state.get(i, (0.0 * g, 0.0 * g))
            m, v = 0.9 * m + 0.1 * g, 0.999 * v + 0.001 * g * g
            self.state[i] = (m, v)
            scale = self.rate / (1.0 - 0.9 ** self.step)
            out.append(p - scale * m / ((v / (1.0 - 0.999 ** self.step)) ** 0.5 + 1e-8))
        return out


def train(x, y, *, width=64, outputs=4, steps=80, kind="bf16", probes=10, rate=0.01, seed=0,
          bits=32, report=print):
    """Trains on x [n, inputs], y [n] (numpy); returns the model, its kernel
    parameters, noise and the history of y^T K^-1 y / n."""
    dtype = TYPES[kind]
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    model = Features(x.shape[1], width, outputs, dtype, gen)
    layers_adam = optim.AdamW(model.parameters(), bits=bits, master=kind != "f32", seed=seed)
    xs = torch.from_numpy(x).to("cuda", dtype)
    ys = torch.from_numpy(y).cuda()
    raw = [np.log(np.array([1.0] * outputs + [1.0, 0.1]))]  # lengthscales, outputscale, noise
    kernel_adam = Adam(3.0 * rate)
    history = []
    for step in range(steps):
        z, tape = model.forward(xs, offset=step * len(x) * width)
        theta = np.exp(raw[0])
        provider = NativeProvider("rbf", True, z.float().cpu().numpy(), theta[:-1],
                                  float(theta[-1]))
        try:
            draws = torch.randn(probes, len(x), generator=gen, device="cuda")
            fit, dz, dtheta = likelihood_gradients(provider, ys, draws)
        finally:
            provider.close()
        history.append(fit / len(x))
        grads = model.backward((dz / len(x)).to(dtype), tape)
        layers_adam.step(grads, rate, step + 1)
        raw = kernel_adam.update(raw, [dtheta / len(x) * theta])
        if report and (step % 10 == 0 or step == steps - 1):
            report(f"step {step:4d}  y K^-1 y / n {history[-1]:.4f}  noise {theta[-1]:.4f}")
    return model, theta, history


def predict(model, theta, x, y, xs, int8=False):
    """Predictive mean at xs (dropout off; int8: by the layers in 8-bit integers, for
    both sides of the kernel)."""
    dtype = model.first[0].dtype
    serve = model.int8() if int8 else lambda a: model.forward(a, rate=0.0)[0]
    z, zs = (serve(torch.from_numpy(a).to("cuda", dtype)).float() for a in (x, xs))
    provider = NativeProvider("rbf", True, z.cpu().numpy(), theta[:-1], float(theta[-1]))
    try:
        alpha = solve(provider, torch.from_numpy(y).cuda()[None])
        return provider.cross_matvec(zs.cpu().numpy(), alpha.cpu().numpy()[0])
    finally:
        provider.close()


def data(n, seed=0):
    """A step along a direction of four inputs: no stationary kernel of the inputs
    fits it well."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((n, 4)).astype(np.float32)
    s = x @ (np.ones(4) / 2.0)
    y = np.sign(s) * (1.0 + 0.3 * np.sin(3.0 * s)) + 0.1 * rng.standard_normal(n)
    return x, y.astype(np.float32)


def main():
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--points", type=int, default=4000)
    parser.add_argument("--steps", type=int, default=80)
    parser.add_argument("--type", choices=sorted(TYPES), default="bf16")
    parser.add_argument("--bits", type=int, choices=(8, 32), default=32, help="AdamW's states")
    parser.add_argument("--int8", action="store_true", help="serve in 8-bit integers")
    args = parser.parse_args()
    x, y = data(args.points + 1000)
    n = args.points
    model, theta, _ = train(x[:n], y[:n], steps=args.steps, kind=args.type, bits=args.bits)
    mean = predict(model, theta, x[:n], y[:n], x[n:], args.int8)
    print(f"test RMSE {np.sqrt(np.mean((mean - y[n:]) ** 2)):.4f} of a spread of {y[n:].std():.4f}")


if __name__ == "__main__":
    main()
