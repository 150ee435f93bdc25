"""The operators of a deep kernel: what they compute, and the work they are measured by.

A deep kernel puts a Gaussian process on learned features: gated layers (two
projections, an activation and their product), layer norms and dropout map the
inputs to the points of the kernel, and the gradient of the marginal likelihood
goes back through the points (the kernel's input gradient) into the layers.
The measured calls are those of one training step and of serving test points.

Sizes: points, dimensions and right-hand sides of bench.py's configurations and
of perf/cases.py (1 to 250 000 points, 1 to 16 kernel dimensions, 1 to 16
columns); feature widths from a handful of columns to 1024, hidden widths to
4096, in float32, bfloat16 and float16, odd ones among them.
"""

import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
ACTIVATIONS = ("silu", "gelu", "sigmoid", "relu")
KERNELS = ("rbf", "matern12", "matern32", "matern52")
OUTPUTSCALE = 1.1


def listed():
    return [
        # the features of one test point before they go into the kernel: latency
        {"name": "norm-serve", "op": "norm", "rows": 1, "width": 256, "type": "f32", "pad": 0,
         "train": False},
        # a training step over features of an odd width that are columns of a wider table
        {"name": "norm-odd", "op": "norm", "rows": 12007, "width": 771, "type": "bf16", "pad": 13,
         "train": True},
        # the features of all points of the benchmark's largest set, forward and backward
        {"name": "norm-large", "op": "norm", "rows": 250000, "width": 256, "type": "f32", "pad": 0,
         "train": True},
        # one test point through a layer: the weights are read once
        {"name": "gated-serve", "op": "gated", "rows": 1, "width": 512, "hidden": 2048,
         "type": "bf16", "act": "silu", "pad": 0, "train": False},
        # a batch of test points
        {"name": "gated-batch", "op": "gated", "rows": 500, "width": 256, "hidden": 1024,
         "type": "f16", "act": "gelu", "pad": 0, "train": False},
        # a training step in the kernel's own type
        {"name": "gated-f32", "op": "gated", "rows": 20000, "width": 256, "hidden": 512,
         "type": "f32", "act": "gelu", "pad": 0, "train": True},
        # one whose sizes fit no tile, on columns of a wider table
        {"name": "gated-odd", "op": "gated", "rows": 12007, "width": 391, "hidden": 1027,
         "type": "bf16", "act": "silu", "pad": 9, "train": True},
        # the largest layer
        {"name": "gated-large", "op": "gated", "rows": 65536, "width": 1024, "hidden": 4096,
         "type": "bf16", "act": "silu", "pad": 0, "train": True},
        # a training step of a middle-sized set, with a residual connection
        {"name": "dropout-mid", "op": "dropout", "rows": 12007, "width": 256, "type": "f32",
         "rate": 0.1, "offset": 0, "residual": True},
        # the largest: the draws' numbers pass 32 bits
        {"name": "dropout-large", "op": "dropout", "rows": 250000, "width": 1024, "type": "bf16",
         "rate": 0.2, "offset": 1 << 34, "residual": True},
        # the gradient of a small model's points (y and 10 probes)
        {"name": "points-small", "op": "points", "kernel": "rbf", "ard": False, "n": 1000, "d": 2,
         "t": 11, "ls": 1.0},
        # that of the gradient step of perf/cases.py
        {"name": "points-large", "op": "points", "kernel": "matern52", "ard": True, "n": 50000,
         "d": 8, "t": 16, "ls": 1.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "gated", "gated", "gated", "dropout", "points", "points"])
    kind = rng.choice(sorted(TYPES))
    pad = rng.choice([0, 0, 1, 8, 13, 64])
    if op == "points":
        return {"op": op, "kernel": rng.choice(KERNELS), "ard": rng.random() < 0.6,
                "n": _log(rng, 300, 30000), "d": rng.randint(1, 16),
                "t": rng.choice([1, 11, 16, rng.randint(2, 16)]),
                "ls": round(math.exp(rng.uniform(math.log(0.3), math.log(2.0))), 3)}
    if op == "gated":
        width, hidden = _log(rng, 16, 1024), _log(rng, 16, 4096)
        # the float32 products cost about eight times the narrower ones
        rows = _log(rng, 1, 8192 if kind == "f32" else 65536)
        if rng.random() < 0.5:  # widths are more often round than not
            width, hidden = 8 * max(1, width // 8), 8 * max(1, hidden // 8)
        return {"op": op, "rows": rows, "width": width, "hidden": hidden, "type": kind,
                "act": rng.choice(ACTIVATIONS), "pad": pad, "train": rng.random() < 0.6}
    width = _log(rng, 8, 8192)
    rows = _log(rng, 1, min(250000, 64000000 // width))
    if op == "norm":
        return {"op": op, "rows": rows, "width": width, "type": kind, "pad": pad,
                "train": rng.random() < 0.6}
    return {"op": op, "rows": rows, "width": width, "type": kind,
            "rate": round(rng.uniform(0.01, 0.6), 3),
            "offset": rng.choice([0, 8 * rng.randint(0, 1 << 40), rng.randint(0, 1 << 40)]),
            "residual": rng.random() < 0.5}


# ---------------------------------------------------------------- inputs

def _points(case, seed):
    """Standardised features, weight columns of the gradient step ([alpha |
    probes] against scaled solves, which leave the probes' rough part) and
    lengthscales that keep typical distances a few lengthscales."""
    rng = np.random.default_rng([20261, int(seed)])
    n, d, t = case["n"], case["d"], case["t"]
    X = rng.standard_normal((n, d), dtype=np.float32)
    R = rng.standard_normal((t, n), dtype=np.float32)
    L = (R + 0.5 * rng.standard_normal((t, n), dtype=np.float32)) * np.float32(5.0 / t)
    base = case["ls"] * max(1.0, math.sqrt(d) / 2)
    ls = base * rng.uniform(0.8, 1.25, size=d) if case["ard"] else np.full(1, base)
    params = np.append(ls, OUTPUTSCALE).astype(np.float32)
    return X, L, R, params


def _inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed) * 7919 + 11)
    kind = TYPES[case.get("type", "f32")]

    def normal(*shape, scale=1.0, shift=0.0):
        a = torch.randn(*shape, device="cuda", generator=gen, dtype=torch.float32)
        return a.mul_(scale).add_(shift)

    if case["op"] == "points":
        X, L, R, params = _points(case, seed)
        return {"X": X, "params": params, "L": torch.from_numpy(L).cuda(),
                "R": torch.from_numpy(R).cuda()}
    rows, width = case["rows"], case["width"]
    if case["op"] == "dropout":
        s = {"x": normal(rows, width).to(kind), "dy": normal(rows, width).to(kind),
             "seed": 0x9E3779B97F4A7C15 ^ (int(seed) * 0x1000003)}
        s["residual"] = normal(rows, width).to(kind) if case["residual"] else None
        return s
    # columns of a wider table where pad is not 0
    x = normal(rows, width + case["pad"])
    if case["op"] == "norm":
        # activations: every row with a level and a spread of its own
        x = x * (0.5 + torch.rand(rows, 1, device="cuda", generator=gen)) + normal(rows, 1)
        return {"x": x.to(kind)[:, :width], "dy": normal(rows, width).to(kind),
                "weight": normal(width, scale=0.1, shift=1.0).to(kind),
                "bias": normal(width, scale=0.1).to(kind)}
    hidden = case["hidden"]
    return {"x": x.to(kind)[:, :width], "dh": normal(rows, hidden).to(kind),
            "w_gate": normal(hidden, width, scale=width ** -0.5).to(kind),
            "w_up": normal(hidden, width, scale=width ** -0.5).to(kind),
            "b_gate": normal(hidden, scale=0.1).to(kind),
            "b_up": normal(hidden, scale=0.1).to(kind)}


class _State(dict):
    def __del__(self):
        try:
            self["provider"].close()
        except Exception:
            pass


def prepare(case, seed):
    s = _State(case=case, **_inputs(case, seed))
    if case["op"] == "points":
        if own:  # the model's handle, which holds its points
            from mojogp_amd._provider import NativeProvider
            s["provider"] = NativeProvider(case["kernel"], case["ard"], s["X"], s["params"], 0.1)
        s["X"] = torch.from_numpy(s["X"]).cuda()
        s["params"] = torch.from_numpy(s["params"]).cuda()
    return s


# ---------------------------------------------------------------- the plain forms, in 32 bits

EPS = 1e-5


def _norm_plain(s, train):
    kind = s["x"].dtype
    x, w = s["x"].float(), s["weight"].float()
    xc = x - x.mean(dim=1, keepdim=True)
    rstd = torch.rsqrt((xc * xc).mean(dim=1, keepdim=True) + EPS)
    xhat = xc * rstd
    y = (xhat * w + s["bias"].float()).to(kind)
    if not train:
        return y
    dy = s["dy"].float()
    g = dy * w
    dx = rstd * (g - g.mean(dim=1, keepdim=True) - xhat * (g * xhat).mean(dim=1, keepdim=True))
    return y, dx.to(kind), (dy * xhat).sum(dim=0).to(kind), dy.sum(dim=0).to(kind)


def _activation(act, g):
    """act(g) and its derivative."""
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-g))
        return g * s, s * (1.0 + g * (1.0 - s))
    if act == "sigmoid":
        s = 1.0 / (1.0 + torch.exp(-g))
        return s, s * (1.0 - s)
    if act == "relu":
        return torch.clamp(g, min=0.0), (g > 0).float()
    cdf = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
    return g * cdf, cdf + g * torch.exp(-0.5 * g * g) / math.sqrt(2.0 * math.pi)


def _gated_plain(s, act, train):
    kind = s["x"].dtype
    x, wg, wu = s["x"].float(), s["w_gate"].float(), s["w_up"].float()
    g = x @ wg.T + s["b_gate"].float()
    u = x @ wu.T + s["b_up"].float()
    a, slope = _activation(act, g)
    h = (a * u).to(kind)
    if not train:
        return h
    dh = s["dh"].float()
    dg, du = dh * u * slope, dh * a
    return (h, (dg @ wg + du @ wu).to(kind), (dg.T @ x).to(kind), (du.T @ x).to(kind),
            dg.sum(dim=0).to(kind), du.sum(dim=0).to(kind))


def _draws(seed, first, count):
    """16-bit draws number first .. first + count - 1 of the stream `seed`:
    draw e is half e % 2 of word (e % 8) / 2 of the Philox4x32-10 block with the
    counter (e / 8, 0) (Salmon et al., "Parallel random numbers: as easy as
    1, 2, 3", 2011) and the seed as its key."""
    low = 0xFFFFFFFF
    block = torch.arange(first // 8, (first + count + 7) // 8, device="cuda")
    c0, c1 = block & low, block >> 32
    c2, c3 = torch.zeros_like(c0), torch.zeros_like(c0)
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (((p1 >> 32) & low) ^ c1 ^ k0, p1 & low,
                          ((p0 >> 32) & low) ^ c3 ^ k1, p0 & low)
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack([c0, c1, c2, c3], dim=1)
    halves = torch.stack([words & 0xFFFF, words >> 16], dim=2).reshape(-1)
    return halves[first % 8:first % 8 + count]


def _dropout_plain(s, rate, offset):
    """Kept where the element's draw is at least round(65536 rate), and scaled
    by the inverse of that share."""
    kind = s["x"].dtype
    x, dy = s["x"].float(), s["dy"].float()
    cut = round(rate * 65536)
    factor = (_draws(s["seed"], offset, x.numel()) >= cut).float().reshape(x.shape)
    factor = factor * (65536.0 / (65536 - cut))
    y = x * factor
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(kind), (dy * factor).to(kind)


def _points_plain(s, kernel, ard):
    """d/dX of sum_ab K(X, X)[a, b] W[a, b], W = L^T R, from differences."""
    X, params = s["X"], s["params"]
    n, d = X.shape
    inv = (1.0 / params[:-1]).expand(d)
    z = X * inv
    r2 = torch.zeros(n, n, device=X.device)
    for q in range(d):
        r2.add_((z[:, q, None] - z[None, :, q]) ** 2)
    if kernel == "rbf":
        h = torch.exp(-0.5 * r2)
    else:
        r = torch.sqrt(r2 + 1e-20)
        u = r * {"matern12": 1.0, "matern32": math.sqrt(3.0), "matern52": math.sqrt(5.0)}[kernel]
        e = torch.exp(-u if kernel == "matern12" and not ard else torch.clamp(-u, min=-20.0))
        h = e / r if kernel == "matern12" else 3.0 * e if kernel == "matern32" else \
            (5.0 / 3.0) * (1.0 + u) * e
    W = s["L"].T @ s["R"]
    h = h * (W + W.T)
    out = torch.empty(n, d, device=X.device)
    for q in range(d):
        out[:, q] = (h * (z[None, :, q] - z[:, q, None])).sum(dim=1) * (inv[q] * params[-1])
    return out


def run(state):
    case, s = state["case"], state
    op = case["op"]
    if not own:
        if op == "norm":
            return _norm_plain(s, case["train"])
        if op == "gated":
            return _gated_plain(s, case["act"], case["train"])
        if op == "dropout":
            return _dropout_plain(s, case["rate"], case["offset"])
        return _points_plain(s, case["kernel"], case["ard"])
    from mojogp_amd import features
    if op == "norm":
        if not case["train"]:
            return features.layer_norm(s["x"], s["weight"], s["bias"], eps=EPS)
        y, saved = features.layer_norm(s["x"], s["weight"], s["bias"], eps=EPS, save=True)
        return (y, *features.layer_norm_backward(s["dy"], s["x"], s["weight"], saved))
    if op == "gated":
        layer = (s["x"], s["w_gate"], s["w_up"], s["b_gate"], s["b_up"])
        h = features.gated_layer(*layer, activation=case["act"])
        if not case["train"]:
            return h
        return (h, *features.gated_layer_backward(s["dh"], *layer, activation=case["act"]))
    if op == "dropout":
        y = features.dropout(s["x"], case["rate"], s["seed"], offset=case["offset"],
                             residual=s["residual"])
        return y, features.dropout_backward(s["dy"], case["rate"], s["seed"],
                                            offset=case["offset"])
    return s["provider"].input_gradient_device(s["L"], s["R"])


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    op = case["op"]
    if op == "points":
        # each unordered pair once: distance, value, both weights, two sums of d
        n, d, t = case["n"], case["d"], case["t"]
        return {"bytes": 4 * (2 * n * d + 2 * n * t),
                "flops": n * (n + 1) / 2 * (3 * d + 12 + 4 * t + 4 * d)}
    size, rows, width = BYTES[case["type"]], case["rows"], case["width"]
    if op == "norm":
        train = case["train"]
        return {"bytes": size * (rows * width * (4 if train else 2) + width * (4 if train else 2)),
                "flops": rows * width * (19 if train else 8)}
    if op == "dropout":
        return {"bytes": size * rows * width * (5 if case["residual"] else 4),
                "flops": 4 * rows * width}
    hidden, train = case["hidden"], case["train"]
    weights = 2 * hidden * (width + 1)
    moved = rows * (width + hidden) * (2 if train else 1) + weights * (2 if train else 1)
    return {"bytes": size * moved, "flops": (12.0 if train else 4.0) * rows * width * hidden}


# ---------------------------------------------------------------- in 64 bits, from the definitions

def _exact_norm(a, train):
    x = a["x"].double().requires_grad_(True)
    w = a["weight"].double().requires_grad_(True)
    b = a["bias"].double().requires_grad_(True)
    var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
    y = (x - mean) / torch.sqrt(var + EPS) * w + b
    if not train:
        return y.detach()
    return (y.detach(), *torch.autograd.grad(y, (x, w, b), a["dy"].double()))


def _exact_gated(a, act, train):
    leaves = [a[k].double().requires_grad_(train)
              for k in ("x", "w_gate", "w_up", "b_gate", "b_up")]
    x, wg, wu, bg, bu = leaves
    g, u = torch.addmm(bg, x, wg.T), torch.addmm(bu, x, wu.T)
    f = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
         "sigmoid": torch.sigmoid, "relu": torch.relu}[act]
    h = f(g) * u
    if not train:
        return h
    return (h.detach(), *torch.autograd.grad(h, leaves, a["dh"].double()))


def _exact_keep(seed, first, count, cut):
    """The kept elements, on the host, a stretch of blocks at a time."""
    mask, shift = np.uint64(0xFFFFFFFF), np.uint64(32)
    out = np.empty(((first + count + 7) // 8 - first // 8) * 8, dtype=bool)
    step = 1 << 16
    for at in range(0, out.size // 8, step):
        stop = min(at + step, out.size // 8)
        number = np.arange(first // 8 + at, first // 8 + stop, dtype=np.uint64)
        x = [number & mask, number >> shift, np.uint64(0), np.uint64(0)]
        key = [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]
        for _ in range(10):
            a, b = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
            x = [(b >> shift) ^ x[1] ^ np.uint64(key[0]), b & mask,
                 (a >> shift) ^ x[3] ^ np.uint64(key[1]), a & mask]
            key = [(key[0] + 0x9E3779B9) & 0xFFFFFFFF, (key[1] + 0xBB67AE85) & 0xFFFFFFFF]
        words = np.stack(x, axis=1).astype("<u4")
        out[at * 8:stop * 8] = words.view("<u2").reshape(-1) >= cut
    return out[first % 8:first % 8 + count]


def _exact_dropout(a, rate, offset):
    x = a["x"].double()
    cut = int(round(rate * 65536))
    keep = torch.from_numpy(_exact_keep(a["seed"], offset, x.numel(), cut)).cuda().view(x.shape)
    factor = torch.where(keep, 65536.0 / (65536 - cut), 0.0)
    y = x * factor + (0.0 if a["residual"] is None else a["residual"].double())
    return y, a["dy"].double() * factor


def _value(kernel, r2, ard):
    if kernel == "rbf":
        return torch.exp(-r2 / 2)
    r = torch.sqrt(r2 + 1e-20)
    if kernel == "matern12":
        return torch.exp(torch.clamp(-r, min=-20.0) if ard else -r)
    if kernel == "matern32":
        u = math.sqrt(3.0) * r
        return (1 + u) * torch.exp(torch.clamp(-u, min=-20.0))
    u = math.sqrt(5.0) * r
    return (1 + u + u * u / 3) * torch.exp(torch.clamp(-u, min=-20.0))


def _exact_points(a, kernel, ard):
    X = torch.from_numpy(a["X"]).cuda().double().requires_grad_(True)
    p = torch.from_numpy(a["params"]).cuda().double()
    L, R = a["L"].double(), a["R"].double()
    step = max(16, (1 << 23) // X.shape[0])
    for i in range(0, X.shape[0], step):
        z = X / p[:-1]
        r2 = 0.0
        for q in range(X.shape[1]):
            r2 = r2 + (z[i:i + step, q, None] - z[None, :, q]) ** 2
        W = L[:, i:i + step].T @ R
        (p[-1] * (W * _value(kernel, r2, ard)).sum()).backward()
    return X.grad


def exact(case, seed):
    a = _inputs(case, seed)
    if case["op"] == "norm":
        return _exact_norm(a, case["train"])
    if case["op"] == "gated":
        return _exact_gated(a, case["act"], case["train"])
    if case["op"] == "dropout":
        return _exact_dropout(a, case["rate"], case["offset"])
    return _exact_points(a, case["kernel"], case["ard"])
