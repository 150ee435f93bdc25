"""Training and serving the layers of a deep kernel: what is computed, and the work it is measured by.

Three operators beside those of perf/operators.py: the AdamW step over all the
layers' parameters at once (with states in 32 or in 8 bits, master copies of
16-bit parameters, and clipping by the norm of all gradients), the group norm
with an activation of features that have positions (grids, series; channels
last), forward and backward, and layers whose trained weights are served in
8-bit integers, with a scale for each test point and each weight row.

Sizes: parameters of layers of 8 to 1024 columns and up to 4096 hidden ones (a
few hundred values to 67 million in 6 to 240 tensors); 1 to 250 000 samples of 1
to 65 536 positions and 1 to 4096 channels; products over 1 to 65 536 points,
in float32, bfloat16 and float16, odd ones among them.
"""

import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
ACTIVATIONS = ("silu", "gelu", "sigmoid", "relu")
EPS = 1e-5        # of the group norm
BETAS = (0.9, 0.999)
ADAM_EPS = 1e-8
DECAY = 0.01
RATE = 1e-3
BLOCK = 256       # values of one scale in the 8-bit states


def listed():
    return [
        # a step on the layers of a small deep kernel (three gated layers of 64 columns): latency
        {"name": "adamw-small", "op": "adamw", "layers": 3, "width": 64, "hidden": 64,
         "type": "bf16", "bits": 32, "master": True, "clip": False, "shift": 0},
        # many tensors of odd sizes at odd addresses, 8-bit states, clipped
        {"name": "adamw-odd", "op": "adamw", "layers": 40, "width": 391, "hidden": 1027,
         "type": "bf16", "bits": 8, "master": True, "clip": True, "shift": 1},
        # the largest layers, in 32 bits throughout, clipped
        {"name": "adamw-large", "op": "adamw", "layers": 8, "width": 1024, "hidden": 4096,
         "type": "f32", "bits": 32, "master": False, "clip": True, "shift": 0},
        # the same with 8-bit states
        {"name": "adamw-8bit", "op": "adamw", "layers": 8, "width": 1024, "hidden": 4096,
         "type": "f32", "bits": 8, "master": False, "clip": False, "shift": 0},
        # the features of one test point: latency
        {"name": "group-serve", "op": "group", "samples": 1, "positions": 1, "channels": 256,
         "groups": 32, "type": "f32", "act": "silu", "pad": 0, "train": False},
        # a training step over the features of all points of a large set, without positions
        {"name": "group-points", "op": "group", "samples": 250000, "positions": 1, "channels": 256,
         "groups": 32, "type": "bf16", "act": "silu", "pad": 0, "train": True},
        # a few series of odd length and groups of 23 channels, columns of a wider table
        {"name": "group-odd", "op": "group", "samples": 13, "positions": 1207, "channels": 391,
         "groups": 17, "type": "f16", "act": "gelu", "pad": 9, "train": True},
        # the largest: features on grids of 64 x 64
        {"name": "group-grid", "op": "group", "samples": 32, "positions": 4096, "channels": 512,
         "groups": 32, "type": "bf16", "act": "silu", "pad": 0, "train": True},
        # one test point through a gated layer: latency, the weights read once
        {"name": "int8-serve", "op": "int8", "rows": 1, "width": 512, "hidden": 2048,
         "type": "bf16", "act": "silu", "gated": True, "pad": 0},
        # a batch of test points through a plain layer
        {"name": "int8-batch", "op": "int8", "rows": 500, "width": 1024, "hidden": 4096,
         "type": "f16", "act": "gelu", "gated": False, "pad": 0},
        # sizes that fit no tile, on columns of a wider table
        {"name": "int8-odd", "op": "int8", "rows": 12007, "width": 391, "hidden": 1027,
         "type": "f32", "act": None, "gated": False, "pad": 9},
        # the largest layer
        {"name": "int8-large", "op": "int8", "rows": 65536, "width": 1024, "hidden": 4096,
         "type": "bf16", "act": "silu", "gated": True, "pad": 0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["adamw", "group", "int8"])
    kind = rng.choice(sorted(TYPES))
    pad = rng.choice([0, 0, 1, 8, 13, 64])
    if op == "adamw":
        layers, width, hidden = _log(rng, 1, 40), _log(rng, 8, 1024), _log(rng, 8, 4096)
        while layers * width * hidden > 30000000:
            layers = (layers + 1) // 2
            hidden = (hidden + 1) // 2
        return {"op": op, "layers": layers, "width": width, "hidden": hidden, "type": kind,
                "bits": rng.choice([8, 32]), "master": kind != "f32" and rng.random() < 0.7,
                "clip": rng.random() < 0.5, "shift": rng.choice([0, 0, 1, 3])}
    if op == "group":
        size, groups = _log(rng, 1, 64), _log(rng, 1, 64)
        if rng.random() < 0.5:  # groups are more often of round sizes than not
            size = 1 << max(2, size.bit_length() - 1)
            groups = 1 << (groups.bit_length() - 1)
        positions = rng.choice([1, _log(rng, 2, 64), _log(rng, 64, 65536)])
        if size * positions < 16:  # (gradients of a few values cancel to nothing)
            size = 16
        channels = size * groups
        positions = min(positions, 48000000 // channels)
        most = max(1, 48000000 // (positions * channels))
        train = rng.random() < 0.6
        # (relu's slope jumps at zero, where some of millions of values come to lie
        # on either side by their last bit)
        return {"op": op, "samples": _log(rng, 1, min(250000, most)), "positions": positions,
                "channels": channels, "groups": groups, "type": kind,
                "act": rng.choice((None, *ACTIVATIONS[:3 if train else 4])), "pad": pad,
                "train": train}
    width, hidden = _log(rng, 16, 1024), _log(rng, 16, 4096)
    if rng.random() < 0.5:
        width, hidden = 16 * max(1, width // 16), 16 * max(1, hidden // 16)
    gated = rng.random() < 0.5
    return {"op": op, "rows": _log(rng, 1, 65536), "width": width, "hidden": hidden, "type": kind,
            "act": rng.choice(ACTIVATIONS if gated else (None, *ACTIVATIONS)), "gated": gated,
            "pad": pad}


# ---------------------------------------------------------------- inputs

def _shapes(case):
    """Parameters of a stack of gated layers with layer norms, in order, and whether
    weight decay takes them (the matrices only)."""
    w, h = case["width"], case["hidden"]
    layer = [((h, w), True), ((h, w), True), ((h,), False), ((h,), False), ((w,), False),
             ((w,), False)]
    return layer * case["layers"]


def _blocks(case):
    """The first block of each parameter, and how many there are: every one
    starts a block of its own."""
    at, starts = 0, []
    for shape, _ in _shapes(case):
        starts.append(at)
        at += (math.prod(shape) + BLOCK - 1) // BLOCK
    return starts, at


def _views(flat, case):
    """The parameters' views of an array of all blocks."""
    return [flat[s * BLOCK:s * BLOCK + math.prod(shape)].view(shape)
            for s, (shape, _) in zip(_blocks(case)[0], _shapes(case))]


def _codes_of(x, mantissa, lowest, top):
    """Codes (in float64, the values they stand for) nearest to x in [0, top]:
    `mantissa` bits, exponents from `lowest` on, evenly spaced below."""
    step = torch.exp2(torch.clamp(torch.floor(torch.log2(x.clamp_min(1e-300))), min=lowest)
                      - mantissa)
    return torch.clamp(torch.round(x / step) * step, max=top)


def _adamw_inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed) * 7919 + 5)
    kind, count = TYPES[case["type"]], _blocks(case)[1]
    n, shift = count * BLOCK, case["shift"]
    inside = torch.zeros(n, device="cuda")  # 1 where a block's place is a parameter's
    for v in _views(inside, case):
        v.fill_(1.0)

    def normal():
        return torch.randn(n, device="cuda", generator=gen)

    def rows(kind, a):  # (an array that may begin at any address)
        flat = torch.zeros(n + shift, device="cuda", dtype=kind)[shift:]
        return flat.copy_(a)

    # of a training run under way: gradients of different sizes by block and by
    # value, means over ten steps and squares over a thousand; unused units have none
    size = torch.exp(torch.randn(count, 1, device="cuda", generator=gen)).mul_(1e-3)
    size = size * (torch.rand(count, 1, device="cuda", generator=gen) > 0.02)
    size = (size * torch.exp(0.7 * normal()).view(count, BLOCK)).view(-1) * inside
    s = {"param": rows(kind, 0.05 * normal() * inside), "grad": rows(kind, size * normal()),
         "decay": torch.zeros(count, 1, device="cuda")}
    m = 0.3 * size * normal()
    v = (size * (0.5 + torch.rand(n, device="cuda", generator=gen))) ** 2
    if case["master"]:
        s["master"] = s["param"].float() * (1.0 + 2.0 ** -10 * (2 * torch.rand(
            n, device="cuda", generator=gen) - 1))
    for start, (shape, decays) in zip(_blocks(case)[0], _shapes(case)):
        if decays:
            s["decay"][start:start + (math.prod(shape) + BLOCK - 1) // BLOCK] = DECAY
    s["step"], s["max_norm"] = 1000, 0.5 if case["clip"] else None
    s["seed"] = 0x9E3779B97F4A7C15 ^ (int(seed) * 0x1000003)
    if case["bits"] == 32:
        s["exp_avg"], s["exp_avg_sq"] = m, v
        return s
    m, v = m.view(count, BLOCK).double(), v.view(count, BLOCK).double()
    ms, vs = (m.abs().amax(1, keepdim=True) / 448).float(), (v.amax(1, keepdim=True) / 1.875).float()
    x = _codes_of(torch.where(ms > 0, m.abs() / ms, 0.0), 3, -6, 448.0) * torch.sign(m)
    s["exp_avg"] = x.to(torch.float8_e4m3fn).view(torch.uint8).view(-1)
    x = _codes_of(torch.where(vs > 0, v / vs, 0.0), 3, -30, 1.875)
    s["exp_avg_sq"] = torch.where(v > 0, _square_codes(x).clamp_min(1), 0).to(torch.uint8).view(-1)
    s["exp_avg_scale"], s["exp_avg_sq_scale"] = ms.view(-1), vs.view(-1)
    return s


def _square_codes(x):
    """Codes of values that the format of the squares has."""
    e = torch.floor(torch.log2(x.clamp_min(1e-300))).clamp_min(-30)
    return torch.round(8 * (x * torch.exp2(-e) - 1) + 8 * (e + 31)).to(torch.int64)


def _inputs(case, seed):
    if case["op"] == "adamw":
        return _adamw_inputs(case, seed)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed) * 7919 + 11)
    kind = TYPES[case["type"]]

    def normal(*shape, scale=1.0, shift=0.0):
        a = torch.randn(*shape, device="cuda", generator=gen, dtype=torch.float32)
        return a.mul_(scale).add_(shift)

    if case["op"] == "group":
        n, l, c = case["samples"], case["positions"], case["channels"]
        x = normal(n, l, c + case["pad"])
        # every sample and channel with a level, every sample with a spread of its own
        x = x * (0.5 + torch.rand(n, 1, 1, device="cuda", generator=gen))
        x += normal(n, 1, c + case["pad"], scale=0.5)
        return {"x": x.to(kind)[..., :c], "dy": normal(n, l, c).to(kind),
                "weight": normal(c, scale=0.1, shift=1.0).to(kind),
                "bias": normal(c, scale=0.1).to(kind)}
    rows, width, hidden = case["rows"], case["width"], case["hidden"]
    x = normal(rows, width + case["pad"])
    x *= torch.exp(normal(rows, 1, scale=0.5)) * torch.exp(normal(1, width + case["pad"], scale=0.4))
    s = {"x": x.to(kind)[:, :width]}
    for name in ("gate", "up")[:2 if case["gated"] else 1]:
        s["w_" + name] = normal(hidden, width, scale=width ** -0.5).to(kind)
        s["b_" + name] = normal(hidden, scale=0.1).to(kind)
    return s


def prepare(case, seed):
    s = dict(_inputs(case, seed), case=case)
    if case["op"] == "adamw":
        s["grads"] = _views(s["grad"], case)
        if own:  # the optimiser, which holds the states
            from mojogp_amd import optim
            s["optimizer"] = optim.AdamW(
                _views(s["param"], case), bits=case["bits"], master=case["master"], betas=BETAS,
                eps=ADAM_EPS, seed=s["seed"],
                weight_decay=[DECAY if d else 0.0 for _, d in _shapes(case)])
            s["optimizer"].load({k: s.pop(k) for k in tuple(s) if k.startswith(("exp_", "master"))})
    if case["op"] == "int8":  # the weights as a server keeps them
        for name in ("gate", "up")[:2 if case["gated"] else 1]:
            w = s.pop("w_" + name)
            if own:
                from mojogp_amd import features
                s["q_" + name] = features.int8_weights(w)
            else:
                codes, s["scale_" + name] = _quantize(w)
                s["q_" + name] = codes.to(torch.int8)
    return s


# ---------------------------------------------------------------- the plain forms

def _words(seed, step, count):
    """Word i % 4 of the Philox4x32-10 block (Salmon et al., "Parallel random
    numbers: as easy as 1, 2, 3", 2011) with counter (i / 4, step) and key seed,
    for value i of the states."""
    low = 0xFFFFFFFF
    block = torch.arange((count + 3) // 4, device="cuda")
    c0, c1 = block & low, block >> 32
    c2, c3 = torch.full_like(c0, step & low), torch.full_like(c0, step >> 32)
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (((p1 >> 32) & low) ^ c1 ^ k0, p1 & low,
                          ((p0 >> 32) & low) ^ c3 ^ k1, p0 & low)
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack([c0, c1, c2, c3], dim=1).reshape(-1)[:count]


def _rounded(x, draw, lowest, most):
    """Codes of values x >= 0 in 64 bits, rounded up with the probability of what
    lies above the code below: 3 mantissa bits, exponents from `lowest` on, evenly
    spaced below; `most` is the largest code."""
    bits = x.view(torch.int64) + ((2 * draw + 1) << 32)
    normal = (bits >> 49) - ((lowest + 1022) << 3)
    small = torch.floor(x * 2.0 ** (3 - lowest) + (2 * draw + 1).double() / 131072).long()
    return torch.where(x < 2.0 ** lowest, small, normal).clamp_max(most)


def _decoded(s, key):
    """The values of 8-bit states, in 64 bits."""
    code = s[key].view(-1, BLOCK)
    if key == "exp_avg":
        x = code.view(torch.float8_e4m3fn).double()
    else:
        code = code.long()
        e = code >> 3
        x = torch.where(e > 0, 8 + (code & 7), code).double() * torch.exp2(
            e.clamp_min(1).double() - 34)
    return x * s[key + "_scale"].double().view(-1, 1)


def _adamw_plain(s, case):
    """In 64 bits where the states are in 8, whose codes are values next to a border."""
    eight = case["bits"] == 8
    wide = torch.float64 if eight else torch.float32
    b1, b2 = BETAS
    g = s["grad"].view(-1, BLOCK).to(wide)
    out = {}
    if case["clip"]:
        norm = torch.sqrt((g.double() * g.double()).sum())
        g = g * torch.clamp(s["max_norm"] / norm, max=1.0).to(wide)
        out["norm"] = norm.float()
    if eight:
        m, v = _decoded(s, "exp_avg"), _decoded(s, "exp_avg_sq")
    else:
        m, v = s["exp_avg"].view(-1, BLOCK), s["exp_avg_sq"].view(-1, BLOCK)
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * (g * g)
    p = s["master" if case["master"] else "param"].view(-1, BLOCK)
    update = (m / (1 - b1 ** s["step"])) / (torch.sqrt(v / (1 - b2 ** s["step"])) + ADAM_EPS)
    p = p.float() * (1 - RATE * s["decay"]) - RATE * update.float()
    if case["master"]:
        out["master"] = s["master"].copy_(p.view(-1))
    out["param"] = s["param"].copy_(p.view(-1))
    if not eight:
        out["exp_avg"] = s["exp_avg"].copy_(m.view(-1))
        out["exp_avg_sq"] = s["exp_avg_sq"].copy_(v.view(-1))
        return out
    word = _words(s["seed"], s["step"], m.numel()).view(-1, BLOCK)
    ms = (m.abs().amax(1, keepdim=True) / 448).float()
    vs = (v.amax(1, keepdim=True) / 1.875).float()
    code = _rounded(torch.where(ms > 0, m.abs() / ms.double(), 0.0), word & 0xFFFF, -6, 126)
    code = torch.where(m < 0, code + 128, code)
    s["exp_avg"].copy_(code.view(-1))
    code = _rounded(torch.where(vs > 0, v / vs.double(), 0.0), word >> 16, -30, 255)
    s["exp_avg_sq"].copy_(torch.where((v > 0) & (vs > 0), code.clamp_min(1), 0).view(-1))
    s["exp_avg_scale"].copy_(ms.view(-1))
    s["exp_avg_sq_scale"].copy_(vs.view(-1))
    out["exp_avg"] = _decoded(s, "exp_avg").float().view(-1)
    out["exp_avg_sq"] = _decoded(s, "exp_avg_sq").float().view(-1)
    return out


def _activation(act, g):
    """act(g) and its derivative."""
    if act is None:
        return g, torch.ones_like(g)
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


def _group_plain(s, case):
    kind = s["x"].dtype
    n, l, c = s["x"].shape
    groups = case["groups"]
    x = s["x"].float().reshape(n, l, groups, c // groups)
    w = s["weight"].float().view(groups, c // groups)
    b = s["bias"].float().view(groups, c // groups)
    xc = x - x.mean(dim=(1, 3), keepdim=True)
    rstd = torch.rsqrt((xc * xc).mean(dim=(1, 3), keepdim=True) + EPS)
    xhat = xc * rstd
    y, slope = _activation(case["act"], xhat * w + b)
    y = y.to(kind).view(n, l, c)
    if not case["train"]:
        return y
    dz = s["dy"].float().view(n, l, groups, c // groups) * slope
    g = dz * w
    dx = rstd * (g - g.mean(dim=(1, 3), keepdim=True)
                 - xhat * (g * xhat).mean(dim=(1, 3), keepdim=True))
    return (y, dx.to(kind).view(n, l, c), (dz * xhat).sum(dim=(0, 1)).to(kind).view(c),
            dz.sum(dim=(0, 1)).to(kind).view(c))


def _quantize(x):
    """Codes -127 .. 127 of each row and its scale: the codes are the row times
    127 / largest, rounded to even (both quotients rounded to 32 bits)."""
    most = x.double().abs().amax(dim=1, keepdim=True)
    some = most > 0
    by = torch.where(some, 127 / most, 0.0).float()
    return torch.round(x.double() * by.double()).float(), (most / 127).float().view(-1)


def _int8_plain(s, case):
    kind = s["x"].dtype
    codes, scale = _quantize(s["x"])

    def project(name):
        sums = codes @ s["q_" + name].float().T
        return sums * scale[:, None] * s["scale_" + name] + s["b_" + name].float()

    y, _ = _activation(case["act"], project("gate"))
    return (y * project("up") if case["gated"] else y).to(kind)


def run(state):
    case, s = state["case"], state
    op = case["op"]
    if not own:
        return {"adamw": _adamw_plain, "group": _group_plain, "int8": _int8_plain}[op](s, case)
    from mojogp_amd import features
    if op == "adamw":
        opt = s["optimizer"]
        norm = opt.step(s["grads"], RATE, s["step"], max_norm=s["max_norm"])
        out = {"param": s["param"], **opt.values()}
        if norm is not None:
            out["norm"] = norm
        return out
    if op == "group":
        layer = (s["x"], case["groups"], s["weight"], s["bias"])
        if not case["train"]:
            return features.group_norm(*layer, eps=EPS, activation=case["act"])
        y, saved = features.group_norm(*layer, eps=EPS, activation=case["act"], save=True)
        return (y, *features.group_norm_backward(s["dy"], *layer, saved, activation=case["act"]))
    if case["gated"]:
        return features.int8_gated_layer(s["x"], s["q_gate"], s["q_up"], s["b_gate"], s["b_up"],
                                         activation=case["act"])
    return features.int8_layer(s["x"], s["q_gate"], s["b_gate"], activation=case["act"])


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    size = BYTES[case["type"]]
    if case["op"] == "adamw":
        n = sum(math.prod(shape) for shape, _ in _shapes(case))
        # parameters and states both ways, gradients once; the values of 8-bit
        # states, which come back as such, are written as well
        per = 3 * size + (8 if case["master"] else 0) + (16 if case["bits"] == 32 else 4 + 8)
        return {"bytes": n * per, "flops": n * (20 if case["bits"] == 32 else 60)}
    if case["op"] == "group":
        n, c = case["samples"] * case["positions"] * case["channels"], case["channels"]
        return {"bytes": size * (n * (4 if case["train"] else 2) + c * (4 if case["train"] else 2)),
                "flops": n * (30 if case["train"] else 12)}
    rows, width, hidden = case["rows"], case["width"], case["hidden"]
    many = 2 if case["gated"] else 1
    return {"bytes": size * (rows * (width + hidden) + many * hidden) + many * hidden * (width + 4),
            "flops": 2.0 * many * rows * width * hidden}


# ---------------------------------------------------------------- in 64 bits, from the definitions

def _limbs(a, b):
    """High and low half of the 64-bit product of 32-bit numbers, from 16-bit limbs."""
    a0, a1, b0, b1 = a & 0xFFFF, a >> 16, b & 0xFFFF, b >> 16
    mid = a1 * b0 + ((a0 * b0) >> 16)
    cross = a0 * b1 + (mid & 0xFFFF)
    return a1 * b1 + (mid >> 16) + (cross >> 16), ((cross & 0xFFFF) << 16) | ((a0 * b0) & 0xFFFF)


def _exact_uniform(seed, step, count):
    """The shares of a code's step that are added before it is cut off, for the
    means and for the squares."""
    x = [torch.arange((count + 3) // 4, device="cuda") & 0xFFFFFFFF,
         torch.arange((count + 3) // 4, device="cuda") >> 32, step & 0xFFFFFFFF, step >> 32]
    x = [torch.as_tensor(v, device="cuda").expand((count + 3) // 4) for v in x]
    key = [seed % (1 << 32), (seed >> 32) % (1 << 32)]
    for _ in range(10):
        h0, l0 = _limbs(x[0], 0xD2511F53)
        h1, l1 = _limbs(x[2], 0xCD9E8D57)
        x = [h1 ^ x[1] ^ key[0], l1, h0 ^ x[3] ^ key[1], l0]
        key = [(key[0] + 0x9E3779B9) % (1 << 32), (key[1] + 0xBB67AE85) % (1 << 32)]
    word = torch.stack(x, dim=-1).reshape(-1)[:count]
    return ((word % 65536).double() + 0.5) / 65536, ((word // 65536).double() + 0.5) / 65536


def _exact_codes(x, share, lowest, top):
    """The value of the format that x, moved up by a share of its step, is cut off to."""
    _, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), torch.clamp(e - 1, min=lowest) - 3)
    return torch.clamp(torch.floor(x / step + share) * step, max=top)


def _exact_states(s, m, v):
    um, uv = (u.view(-1, BLOCK) for u in _exact_uniform(s["seed"], s["step"], m.numel()))
    ms = (m.abs().amax(1, keepdim=True) / 448).float().double()
    vs = (v.amax(1, keepdim=True) / 1.875).float().double()
    x = _exact_codes(torch.nan_to_num(m.abs() / ms), um, -6, 448.0)
    y = _exact_codes(torch.nan_to_num(v / vs), uv, -30, 1.875)
    y = torch.where(v > 0, y.clamp_min(2.0 ** -33), 0.0)
    return torch.sign(m) * x * ms, y * vs


def _exact_adamw(s, case):
    g = s["grad"].double().view(-1, BLOCK)
    out = {}
    if case["clip"]:
        out["norm"] = torch.linalg.vector_norm(g)
        if out["norm"] > s["max_norm"]:
            g = g * (s["max_norm"] / out["norm"])
    if case["bits"] == 8:
        m = (s["exp_avg"].view(torch.float8_e4m3fn).double().view(-1, BLOCK)
             * s["exp_avg_scale"].double()[:, None])
        at = torch.arange(256, device="cuda", dtype=torch.float64)  # values of all codes
        e, f = torch.floor(at / 8), at % 8
        table = torch.where(e > 0, torch.ldexp(1 + f / 8, e - 31), torch.ldexp(f / 8, -30 + 0 * e))
        v = table[s["exp_avg_sq"].long()].view(-1, BLOCK) * s["exp_avg_sq_scale"].double()[:, None]
    else:
        m, v = (s[k].double().view(-1, BLOCK) for k in ("exp_avg", "exp_avg_sq"))
    m = torch.lerp(g, m, BETAS[0])
    v = torch.lerp(g.square(), v, BETAS[1])
    t = s["step"]
    p = s["master" if case["master"] else "param"].double().view(-1, BLOCK)
    p = p - RATE * s["decay"].double() * p
    p = p - RATE * (m / -math.expm1(t * math.log(BETAS[0]))) / (
        (v / -math.expm1(t * math.log(BETAS[1]))).sqrt() + ADAM_EPS)
    out["param"] = p.view(-1)
    if case["master"]:
        out["master"] = p.view(-1)
    if case["bits"] == 8:
        m, v = _exact_states(s, m, v)
    return {**out, "exp_avg": m.reshape(-1), "exp_avg_sq": v.reshape(-1)}


def _exact_group(a, case):
    n, l, c = a["x"].shape
    x, w, b = (a[k].double().requires_grad_(True) for k in ("x", "weight", "bias"))
    parts = x.unflatten(2, (case["groups"], -1))
    var, mean = torch.var_mean(parts, dim=(1, 3), correction=0, keepdim=True)
    z = ((parts - mean) / torch.sqrt(var + EPS)).flatten(2) * w + b
    f = {None: lambda t: t, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
         "sigmoid": torch.sigmoid, "relu": torch.relu}[case["act"]]
    y = f(z)
    if not case["train"]:
        return y.detach()
    return (y.detach(), *torch.autograd.grad(y, (x, w, b), a["dy"].double()))


def _exact_int8(a, case):
    def codes(t):
        t = t.double()
        most = torch.linalg.vector_norm(t, ord=math.inf, dim=1)
        by = torch.nan_to_num(127.0 / most, posinf=0.0).float().double()
        return torch.round(t * by[:, None]), (most / 127.0).float().double()

    def project(name):
        w, sw = codes(a["w_" + name])
        # products in 32 bits over 512 columns are whole numbers below 2^23: exact
        total = 0.0
        for k in range(0, x.shape[1], 512):
            total = total + (x[:, k:k + 512].float() @ w[:, k:k + 512].float().T).double()
        return torch.addcmul(a["b_" + name].double(), total, sx[:, None] * sw)

    x, sx = codes(a["x"])
    f = {None: lambda t: t, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
         "sigmoid": torch.sigmoid, "relu": torch.relu}[case["act"]]
    y = f(project("gate"))
    return y * project("up") if case["gated"] else y


def exact(case, seed):
    a = _inputs(case, seed)
    return {"adamw": _exact_adamw, "group": _exact_group, "int8": _exact_int8}[case["op"]](a, case)
