"""The AdamW step on the device against its float64 formulas.

Tolerances.  32-bit states: the factor, the product, and the fused addition round by
2^-24 each: a mean is within 4 * 2^-24 of |b1 m| + |(1 - b1) g|, a square (one more
product) within 5 * 2^-24 of its value.  The step m c1 / (sqrt(v c2) + eps) adds, beside
half of v's and all of m's, the roundings of c1, c2, two products, a root and a
reciprocal of one last place each (2^-23), the sum, the product and the rate: below
16 * 2^-24 of (|b1 m| + |(1 - b1) g|) c1 / (sqrt(v c2) + eps) times the rate; the
parameter is rounded twice (keep and the sum).  8-bit states: codes are equal, the
step as above from means that are rounded once."""

import numpy as np
import pytest
import torch

from mojogp_amd import _lib, optim
from oracle import optim as oo

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
UNIT = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
U = 2.0 ** -24
BETAS, EPS = (0.9, 0.99), 1e-8
SHAPES = [(1,), (3,), (255,), (256,), (257,), (2047,), (2048,), (2049,), (33, 67), (0, 5), (3, 1, 5),
          (4100,)]


def _host(t):
    return t.detach().double().cpu().numpy().ravel()


def _tensors(rng, shapes, kind, scale, shift=1):
    """Tensors at odd places of one array with NaN between them."""
    flat = torch.full((sum(int(np.prod(s)) + 3 for s in shapes) + shift,), float("nan"),
                      device="cuda", dtype=kind)
    out, at = [], shift
    for s in shapes:
        n = int(np.prod(s))
        v = flat[at:at + n].view(s)
        v.copy_(torch.from_numpy(scale * rng.normal(size=s)))
        out.append(v)
        at += n + 3
    return out, flat


def _padded(parts):
    out = []
    for a in parts:
        out.append(np.concatenate([a, np.zeros(-len(a) % 256)]))
    return np.concatenate(out)


class Oracle:
    """The states of an optimiser, stepped in float64 from what the device holds."""

    def __init__(self, opt, decay):
        self.opt, self.decay = opt, decay
        self.inside = _padded([np.ones(p.numel()) for p in opt.params]) > 0

    def read(self):
        o = self.opt
        if o.bits == 8:
            m = oo.decode(o.exp_avg.cpu().numpy(), o.exp_avg_scale.cpu().numpy(), True)
            v = oo.decode(o.exp_avg_sq.cpu().numpy(), o.exp_avg_sq_scale.cpu().numpy(), False)
        else:
            m, v = _host(o.exp_avg), _host(o.exp_avg_sq)
        return _padded([_host(p) for p in o.params]), m, v, \
            None if o.master is None else _host(o.master)

    def check(self, before, grads, rate, step, factor=1.0, seed=0, kind="f32"):
        p, m, v, master = before
        live = _padded([np.full(q.numel(), g is not None) for q, g in
                        zip(self.opt.params, grads)]).astype(bool)
        g = _padded([np.zeros(q.numel()) if x is None else _host(x)
                     for q, x in zip(self.opt.params, grads)]) * factor
        nm, nv = oo.moments(m, v, g, BETAS)
        old = p if master is None else master
        decay = _padded([np.full(q.numel(), d) for q, d in zip(self.opt.params, self.decay)])
        want = oo.update(old, nm, nv, rate, step, BETAS, EPS, decay)
        size = BETAS[0] * np.abs(m) + (1 - BETAS[0]) * np.abs(g)
        c1, c2 = 1 - BETAS[0] ** step, 1 - BETAS[1] ** step
        tol = 16 * U * rate * size / c1 / (np.sqrt(nv / c2) + EPS) + 2 * U * np.abs(old) \
            + U * np.abs(want)
        p1, m1, v1, master1 = self.read()
        at = live & self.inside
        new = p1 if master is None else master1
        assert (np.abs(new - want)[at] <= (tol + (UNIT[kind] * np.abs(want) + 2.0 ** -25 if master
                                                  is None and kind != "f32" else 0.0))[at]).all()
        if master is not None:  # the parameters are their roundings
            for q, w in zip(self.opt.params, self.opt.split(self.opt.master)):
                assert torch.equal(q, w.to(q.dtype))
        for a, b in ((p, p1), (m, m1), (v, v1)):
            assert np.array_equal(a[~live & self.inside], b[~live & self.inside])
        if self.opt.bits == 32:
            assert (np.abs(m1 - nm)[at] <= 4 * U * size[at] + 1e-38).all()
            assert (np.abs(v1 - nv)[at] <= 5 * U * nv[at] + 1e-38).all()
            return
        word = oo.words(seed, step, len(nm))
        block = live.reshape(-1, 256)[:, 0]
        for x, draw, signed, codes, scales in (
                (nm, word & 0xFFFF, True, self.opt.exp_avg, self.opt.exp_avg_scale),
                (nv, word >> 16, False, self.opt.exp_avg_sq, self.opt.exp_avg_sq_scale)):
            code, scale = oo.encode(np.where(self.inside, x, 0.0), draw, signed)
            code, got = code.reshape(-1, 256), codes.cpu().numpy().reshape(-1, 256)
            if signed:  # a rounded-off negative value keeps its sign
                code, got = (np.where(c == 128, 0, c) for c in (code, got))
            assert np.array_equal(code[block], got[block])
            assert np.array_equal(scale[block], scales.cpu().numpy()[block])


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("kind, master, wide", [("f32", False, False), ("bf16", False, False),
                                                ("bf16", True, False), ("bf16", True, True),
                                                ("f16", False, True), ("f16", True, False)])
def test_steps(bits, kind, master, wide):
    rng = np.random.default_rng(bits + len(kind))
    params, flat = _tensors(rng, SHAPES, TYPES[kind], 0.1)
    between = torch.isnan(flat)
    decay = [0.1 * (i % 3) for i in range(len(SHAPES))]
    opt = optim.AdamW(params, bits=bits, master=master, betas=BETAS, eps=EPS, weight_decay=decay,
                      seed=(1 << 63) + 5)
    o = Oracle(opt, decay)
    for step in (1, 2, 3):
        grads, _ = _tensors(rng, SHAPES, torch.float32 if wide else TYPES[kind], 10.0 ** -step, 3)
        if step == 2:
            grads[4] = grads[8] = None
        if step == 3:  # a unit without gradients
            grads[7].zero_()
        before = o.read()
        assert opt.step(grads, 0.01, step) is None
        o.check(before, grads, 0.01, step, seed=(1 << 63) + 5, kind=kind)
    assert torch.equal(torch.isnan(flat), between)


@pytest.mark.parametrize("bits", [32, 8])
def test_clipping_over_many_tensors(bits):
    """More tensors than one launch takes, some without gradients, clipped or not."""
    rng = np.random.default_rng(9)
    shapes = [(1 + 37 * i % 401,) for i in range(1003)]
    params, _ = _tensors(rng, shapes, torch.float32, 1.0)
    opt = optim.AdamW(params, bits=bits, betas=BETAS, eps=EPS, seed=3)
    o = Oracle(opt, [0.0] * len(shapes))
    for step, limit in ((1, 0.5), (2, 1e9), (3, None)):
        grads, _ = _tensors(rng, shapes, torch.float32, 0.3)
        grads[17] = grads[402] = None
        scaled = [0.25 * _host(g) for g in grads if g is not None]
        norm, factor = oo.clip(scaled, np.inf if limit is None else limit)
        before = o.read()
        got = opt.step(grads, 0.01, step, max_norm=limit, norm=True, grad_scale=0.25)
        # summed in 64 bits, rounded once
        assert got.dtype == torch.float32 and got.shape == ()
        assert abs(float(got) - norm) <= 1.01 * U * norm
        o.check(before, grads, 0.01, step, factor=0.25 * factor, seed=3)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_a_norm_that_is_not_finite_changes_nothing(bits, bad):
    rng = np.random.default_rng(2)
    params, flat = _tensors(rng, [(300,), (40, 40)], torch.float32, 1.0)
    opt = optim.AdamW(params, bits=bits, betas=BETAS, eps=EPS)
    grads, _ = _tensors(rng, [(300,), (40, 40)], torch.float32, 1.0)
    opt.step(grads, 0.01, 1)
    kept = {k: t.clone() for k, t in opt.state().items()}
    old = flat.clone()
    grads[1][3, 7] = bad
    norm = opt.step(grads, 0.01, 2, max_norm=1.0)
    assert not torch.isfinite(norm)
    assert torch.equal(flat.nan_to_num(7.0), old.nan_to_num(7.0))
    for k, t in opt.state().items():
        assert torch.equal(t, kept[k])


@pytest.mark.parametrize("step, rate", [(0, 0.1), (-3, 0.1), (1, float("nan")), (1, float("inf")),
                                        (1, -0.1)])
@pytest.mark.parametrize("bits", [32, 8])
def test_device_numbers_that_are_refused_on_the_host_change_nothing(bits, step, rate):
    p = torch.ones(300, device="cuda")
    opt = optim.AdamW([p], bits=bits)
    g = torch.ones_like(p)
    opt.step([g], torch.full((), rate, device="cuda"), torch.full((), step, device="cuda"))
    assert torch.equal(p, torch.ones_like(p))
    assert all(not t.any() for t in opt.state().values())


def test_a_norm_past_float32_changes_nothing():
    """Of finite gradients: 2^126 times the root of 300."""
    p = torch.ones(300, device="cuda")
    opt = optim.AdamW([p])
    norm = opt.step([torch.full_like(p, 2.0 ** 126)], 0.1, 1, max_norm=1.0)
    assert torch.isinf(norm) and torch.equal(p, torch.ones_like(p)) and not opt.exp_avg.any()


def test_large_and_small_gradients_norm():
    """Squares beyond and below fp32."""
    p = torch.zeros(1000, device="cuda")
    opt = optim.AdamW([p])
    for size in (1e30, 1e-30):
        g = torch.full((1000,), size, device="cuda")
        norm = opt.step([g], 0.0, 1, norm=True)
        want = float(g[0].double()) * 1000 ** 0.5
        assert abs(float(norm) - want) <= 1e-6 * want


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_eight_bit_blocks_that_are_not_finite(bad):
    """Without a norm a value that is not finite spoils its block's states and no other."""
    rng = np.random.default_rng(4)
    (p,), _ = _tensors(rng, [(1024,)], torch.float32, 1.0)
    (q,), _ = _tensors(rng, [(1024,)], torch.float32, 1.0)
    (g,), _ = _tensors(rng, [(1024,)], torch.float32, 1.0)
    q.copy_(p)
    one, two = (optim.AdamW([t], bits=8, betas=BETAS) for t in (p, q))
    two.step([g.clone()], 0.01, 1)
    g[300] = bad
    one.step([g], 0.01, 1)
    ok = torch.ones(1024, dtype=torch.bool, device="cuda")
    ok[256:512] = False
    a, b = one.values(), two.values()
    for k in a:
        assert torch.equal(a[k][ok], b[k][ok]) and torch.isnan(a[k][~ok]).any()
    ok[256:512] = True
    ok[300] = False
    assert torch.equal(p[ok], q[ok]) and not torch.isfinite(p[300])


def test_tiny_states_become_zero():
    """Squares below 2^-120 are held as zeros, and a v above zero never is within
    a block of others."""
    p = torch.zeros(512, device="cuda")
    g = torch.full((512,), 1e-20, device="cuda")
    g[256:] = 1e-6
    g[256] = 1.0
    opt = optim.AdamW([p], bits=8, betas=BETAS, eps=EPS)
    for step in range(1, 4):
        opt.step([g], 1e-3, step)
    v = opt.values()["exp_avg_sq"]
    assert not v[:256].any() and (v[257:] > 0).all()
    # m's smallest code over v's: of the order of one, not of 1 / eps
    assert float(p.abs().max()) < 3 * 1e-3 * 3


def test_eight_bit_means_are_unbiased():
    """A constant gradient: m and v approach it and its square as the formulas do.
    The rounding of v is a walk with steps of variance f (1 - f) (v / 8)^2 / v^2, f
    = (1 - b2) 8 at most, remembered for 1 / (1 - b2) steps: below 0.08 (1/8)^2 100 =
    0.13 of v^2 in variance; the mean of 65536 values is within 5 sqrt(0.13 / 65536) =
    0.7 %.  m: steps of variance 1 / 4 (1 / 8)^2 remembered for 5: 0.02, 0.3 %."""
    n = 65536
    p = torch.zeros(n, device="cuda")
    g = torch.linspace(0.5, 1.0, n, device="cuda")
    opt = optim.AdamW([p], bits=8, betas=BETAS, eps=EPS, seed=11)
    for step in range(1, 301):
        opt.step([g], 0.0, step)
    got = opt.values()
    for key, beta, want, tol in (("exp_avg", BETAS[0], g, 0.003),
                                 ("exp_avg_sq", BETAS[1], g * g, 0.007)):
        ratio = (got[key] / (want * (1 - beta ** 300))).double().mean()
        assert abs(float(ratio) - 1.0) <= tol


@pytest.mark.parametrize("bits", [32, 8])
def test_graph_replays(bits):
    """A step recorded with its rate, number and norm on the device, replayed with
    other work between, against the same steps by single calls."""
    rng = np.random.default_rng(6)
    shapes = [(700,), (129, 33), (5,)]
    params, _ = _tensors(rng, shapes, torch.bfloat16, 0.1)
    others = [p.clone() for p in params]
    grads = [torch.zeros_like(p) for p in params]
    kw = dict(bits=bits, master=True, betas=BETAS, eps=EPS, weight_decay=0.1, seed=8)
    one, two = optim.AdamW(params, **kw), optim.AdamW(others, **kw)
    rate = torch.zeros((), device="cuda")
    step = torch.ones((), device="cuda", dtype=torch.int64)
    before = [p.clone() for p in params]
    state = {k: t.clone() for k, t in one.state().items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        one.step(grads, rate, step, max_norm=0.3)
    torch.cuda.current_stream().wait_stream(side)
    for p, q in zip(params, before):
        p.copy_(q)
    one.load(state)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = one.step(grads, rate, step, max_norm=0.3)
    for t in range(1, 6):
        for g in grads:
            g.copy_(torch.from_numpy(rng.normal(size=tuple(g.shape))))
        rate.fill_(0.01 / t)
        step.fill_(t)
        graph.replay()
        torch.ones(1000, device="cuda").mul_(2).sum().item()
        want = two.step(grads, float(rate), t, max_norm=0.3)
        assert torch.equal(norm, want)
        for p, q in zip(params, others):
            assert torch.equal(p, q)
        for k, s in two.state().items():
            assert torch.equal(one.state()[k], s)


def test_state_moves_on_to_another_optimizer():
    rng = np.random.default_rng(12)
    params, _ = _tensors(rng, [(500,), (20, 30)], torch.bfloat16, 0.1)
    others = [p.clone() for p in params]
    kw = dict(bits=8, master=True, betas=BETAS, seed=2)
    one = optim.AdamW(params, **kw)
    for t in (1, 2):
        one.step(_tensors(rng, [(500,), (20, 30)], torch.bfloat16, 1.0)[0], 0.01, t)
    for p, q in zip(params, others):
        q.copy_(p)
    two = optim.AdamW(others, **kw)
    two.load(one.state())
    grads, _ = _tensors(rng, [(500,), (20, 30)], torch.bfloat16, 1.0)
    for opt in (one, two):
        opt.step(grads, 0.01, 3)
    for p, q in zip(params, others):
        assert torch.equal(p, q)
    for k, t in one.state().items():
        assert torch.equal(two.state()[k], t)
    with pytest.raises(ValueError, match="states"):
        two.load({"exp_avg": one.exp_avg})
    with pytest.raises(ValueError, match="exp_avg must be"):
        two.load({**one.state(), "exp_avg": one.exp_avg[:-1]})


def test_refusals():
    p = torch.zeros(40, 30, device="cuda")
    g = torch.zeros_like(p)
    for bad, err in (([p, p], _lib.NativeCallError), ([p.t()], ValueError),
                     ([p, p.to(torch.bfloat16)], TypeError),
                     ([p.clone().requires_grad_()], ValueError)):
        with pytest.raises(err):
            optim.AdamW(bad)
    for kw in ({"bits": 16}, {"master": True}, {"weight_decay": -1.0}, {"betas": (1.0, 0.9)}):
        with pytest.raises(_lib.NativeCallError):
            optim.AdamW([p], **kw)
    for kw in ({"weight_decay": [0.1, 0.1]}, {"seed": -1}, {"seed": 0.5}):
        with pytest.raises(ValueError):
            optim.AdamW([p], **kw)
    opt = optim.AdamW([p])
    for grads, err in (([], ValueError), ([g, g], ValueError), ([g[:-1]], ValueError),
                       ([g.t()], ValueError), ([g.half()], TypeError), ([g.cpu()], ValueError),
                       ([p], _lib.NativeCallError), ([g.clone().requires_grad_()], ValueError)):
        with pytest.raises(err):
            opt.step(grads, 0.1, 1)
    for rate, step in ((-0.1, 1), (float("nan"), 1), (0.1, 0), (0.1, 1.5),
                       (torch.zeros(2, device="cuda"), 1), (0.1, torch.ones(1, device="cuda")),
                       (torch.zeros(1), 1)):
        with pytest.raises((ValueError, TypeError)):
            opt.step([g], rate, step)
    for kw in ({"max_norm": 0.0}, {"max_norm": float("nan")}, {"grad_scale": 0.0}):
        with pytest.raises(_lib.NativeCallError):
            opt.step([g], 0.1, 1, **kw)
    opt.step([None], 0.1, 1)
    p.data = torch.zeros(40, 30, device="cuda")
    with pytest.raises(ValueError, match="memory"):
        opt.step([g], 0.1, 1)
    opt.close()
    with pytest.raises(ValueError, match="closed"):
        opt.step([g], 0.1, 1)


def test_no_grad_parameters():
    """Leaves of a graph are stepped under no_grad."""
    p = torch.ones(10, device="cuda", requires_grad=True)
    with torch.no_grad():
        opt = optim.AdamW([p], eps=EPS)
        opt.step([torch.ones(10, device="cuda")], 0.5, 1)
    assert torch.allclose(p.detach(), torch.full((10,), 0.5, device="cuda"))
    with pytest.raises(ValueError, match="requires a gradient"):
        opt.step([torch.ones(10, device="cuda")], 0.5, 2)
