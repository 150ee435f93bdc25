"""The group norm on the device against its float64 formulas.

Tolerances, on the 2-norm of the difference over that of the result: one rounding to
the type (unit roundoff u), and fp32 statistics and sums, 2^-24 sqrt(n) for up to n =
20000 terms of either sign a sum and the activations' polynomials: F32 = 1e-5.  dx is
the difference of rstd w dz and its means: its fp32 errors are relative to that."""

import numpy as np
import pytest
import torch

from mojogp_amd import _lib, features
from oracle import layers as ol

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
UNIT = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
F32 = 1e-5
ACTS = (None, "silu", "gelu", "sigmoid", "relu")


def _dev(a, kind, pad=0, shift=0):
    """Rounded to `kind` on the device, in rows of a wider table of NaN."""
    a = np.asarray(a, np.float64)
    if a.ndim == 1:
        return torch.from_numpy(a).to("cuda", TYPES[kind])
    wide = torch.full((*a.shape[:-1], a.shape[-1] + pad), float("nan"), dtype=TYPES[kind],
                      device="cuda")
    view = wide[..., shift:shift + a.shape[-1]]
    view.copy_(torch.from_numpy(a))
    return view


def _host(t):
    return t.double().cpu().numpy()


def _near(got, want, tol, of=None):
    assert tuple(got.shape) == want.shape
    size = np.linalg.norm(want if of is None else of)
    assert np.linalg.norm(_host(got) - want) <= tol * size + 1e-30


def _check(x, dy, groups, w, b, act, kind):
    y, saved = features.group_norm(x, groups, w, b, activation=act, save=True)
    assert torch.equal(y, features.group_norm(x, groups, w, b, activation=act))
    dx, dw, db = features.group_norm_backward(dy, x, groups, w, b, saved, activation=act)
    X, DY = _host(x), _host(dy)
    W, B = (None if p is None else _host(p) for p in (w, b))
    u = UNIT[kind] + F32
    _near(y, ol.group_norm(X, groups, W, B, act), u)
    rx, rw, rb = ol.group_norm_backward(DY, X, groups, W, B, act)
    c = X.shape[-1] // groups
    g = X.reshape(X.shape[0], -1, groups, c)
    rstd = 1 / np.sqrt(g.var(axis=(1, 3), keepdims=True) + 1e-5)
    scale = (rstd * (DY * (1.0 if W is None else W)).reshape(g.shape))
    assert np.linalg.norm(_host(dx) - rx) <= \
        UNIT[kind] * np.linalg.norm(rx) + F32 * np.linalg.norm(scale)
    assert y.dtype == dx.dtype == x.dtype
    rows = X.size // X.shape[-1]
    for got, want, p in ((dw, rw, w), (db, rb, b)):
        assert (got is None) == (p is None)
        if got is not None:
            pk = next(k for k in TYPES if TYPES[k] == p.dtype)
            assert got.dtype == p.dtype and tuple(got.shape) == want.shape
            # sums of `rows` terms of the size of dy: also where they cancel
            assert np.linalg.norm(_host(got) - want) <= (UNIT[pk] + F32) * np.linalg.norm(want) \
                + F32 * np.sqrt(rows * want.size)
    return y, dx


SHAPES = [
    # single positions: groups within a vector, of vectors, of neither; many of them
    (1, 1, 256, 32, 0), (3, 1, 1, 1, 0), (5, 1, 12, 3, 0), (700, 1, 64, 32, 0), (33, 1, 96, 12, 5),
    (40, 1, 512, 2, 0), (9, 1, 391, 17, 3), (513, 1, 24, 3, 0), (3, 1, 4096, 4, 0),
    (2, 1, 5000, 8, 0), (5000, 1, 33, 11, 1), (2100, 1, 16, 16, 0),
    # few positions
    (7, 2, 40, 5, 0), (130, 3, 24, 2, 1), (65, 9, 7, 7, 0), (3, 50, 96, 3, 0), (4, 130, 10, 2, 0),
    (2, 600, 30, 10, 0), (300, 5, 256, 32, 0),
    # long ones, which go in stretches, and channels beyond one block of columns
    (2, 3000, 30, 10, 0), (1, 5001, 256, 32, 0), (3, 1207, 391, 17, 9), (2, 900, 2056, 8, 0),
    (1, 40000, 8, 2, 0), (1, 20, 8200, 5, 0), (2, 30000, 1, 1, 0), (1, 2, 20000, 1, 7),
]


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("n, l, c, groups, pad", SHAPES)
def test_group_norm(kind, n, l, c, groups, pad):
    rng = np.random.default_rng(n + 7 * l + 31 * c)
    act = ACTS[(n + c) % 4]  # (not relu, whose slope jumps)
    x = rng.normal(size=(n, l, c)) * rng.uniform(0.5, 2, (n, 1, 1)) + rng.normal(size=(n, 1, c))
    x = _dev(x, kind, pad, min(pad, 1))
    w, b = _dev(1 + 0.2 * rng.normal(size=c), kind), _dev(0.3 * rng.normal(size=c), kind)
    dy = _dev(rng.normal(size=(n, l, c)), kind, pad)
    _check(x, dy, groups, w, b, act, kind)


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("n, l, c, groups, pad", [
    # a group a channel, to the most that a workgroup holds
    (300, 5, 4096, 4096, 0), (260, 2, 4090, 4090, 0), (70, 12, 100, 100, 0), (50, 28, 14, 14, 0),
    # groups that cut vectors, in slots of one row and of several
    (400, 34, 60, 5, 0), (20, 60, 300, 25, 0), (9, 100, 96, 8, 3), (30, 11, 54, 18, 1),
    (33, 8, 1001, 7, 0),
])
def test_groups_that_cut_vectors(kind, n, l, c, groups, pad):
    rng = np.random.default_rng(n + l + c)
    x = rng.normal(size=(n, l, c)) * rng.uniform(0.5, 2, (n, 1, 1)) + rng.normal(size=(n, 1, c))
    x = _dev(x, kind, pad, min(pad, 1))
    w, b = _dev(1 + 0.2 * rng.normal(size=c), kind), _dev(0.3 * rng.normal(size=c), kind)
    _check(x, _dev(rng.normal(size=(n, l, c)), kind, pad), groups, w, b, ACTS[(n + c) % 4], kind)


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("shape", [(40, 1, 64), (6, 30, 48), (2, 2500, 24)])
def test_activations(kind, act, shape):
    rng = np.random.default_rng(shape[1])
    x = rng.normal(size=shape)
    if act == "relu":  # no value close to the jump of the slope: rows of +-1
        x = np.sign(x) + 0.01 * rng.normal(size=shape)
    x, dy = _dev(x, kind), _dev(rng.normal(size=shape), kind)
    w, b = torch.ones(shape[-1], device="cuda"), torch.zeros(shape[-1], device="cuda")
    _check(x, dy, 4, w, b, act, kind)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("which", [(True, True), (True, False), (False, True), (False, False)])
def test_parameters(kind, which):
    """float32 parameters of 16-bit features, and none."""
    rng = np.random.default_rng(3)
    for shape in ((50, 1, 32), (4, 20, 30), (1, 4000, 40)):
        x, dy = _dev(rng.normal(size=shape), kind), _dev(rng.normal(size=shape), kind)
        w, b = (_dev(rng.normal(size=shape[-1]), "f32") if f else None for f in which)
        _check(x, dy, 2, w, b, "silu", kind)


def test_shapes_of_positions():
    rng = np.random.default_rng(4)
    x, dy = (_dev(rng.normal(size=(3, 4, 5, 24)), "f32") for _ in range(2))
    w, b = (_dev(rng.normal(size=24), "f32") for _ in range(2))
    y, saved = features.group_norm(x, 6, w, b, save=True)
    flat, _ = features.group_norm(x.view(3, 20, 24), 6, w, b, save=True)
    assert torch.equal(y.view(3, 20, 24), flat) and saved.shape == (3, 6, 2)
    got = features.group_norm_backward(dy, x, 6, w, b, saved)
    want = features.group_norm_backward(dy.view(3, 20, 24), x.view(3, 20, 24), 6, w, b, saved)
    assert torch.equal(got[0].view(3, 20, 24), want[0]) and torch.equal(got[1], want[1])
    one = features.group_norm(x[0, 0], 6, w, b)  # samples without positions
    assert torch.equal(one, features.group_norm(x[0, 0].unsqueeze(1), 6, w, b).squeeze(1))


@pytest.mark.parametrize("shape", [(5, 24), (4, 0, 24), (0, 24), (0, 7, 24)])
def test_empty(shape):
    x = torch.zeros(shape, device="cuda")
    w, b = torch.ones(24, device="cuda"), torch.ones(24, device="cuda")
    y, saved = features.group_norm(x, 3, w, b, save=True)
    assert y.shape == shape and saved.shape == (shape[0], 3, 2)
    dx, dw, db = features.group_norm_backward(x, x, 3, w, b, saved)
    assert dx.shape == shape and not dw.any() and not db.any()
    assert torch.equal(y, torch.ones_like(y))  # a constant group: the bias


@pytest.mark.parametrize("shape", [(3, 1, 64), (3, 40, 64), (2, 4000, 64)])
def test_levels_and_values_that_are_not_finite(shape):
    """A level far above the spread costs its own rounding alone; infinities and NaN
    spoil their sample's group and no other."""
    rng = np.random.default_rng(8)
    x = rng.normal(size=shape)
    x[0] += 4096.0
    t = _dev(x, "f32")
    clean, saved = features.group_norm(t, 8, save=True)
    want = ol.group_norm(_host(t), 8)
    # the mean's rounding, 2^-24 4096 of a spread of one, and as much of the differences
    assert np.abs(_host(clean[0]) - want[0]).max() <= 4096 * 2.0 ** -23 * max(
        1.0, float(saved[0, :, 1].max()))
    dy = _dev(rng.normal(size=shape), "f32")
    dx, _, _ = features.group_norm_backward(dy, t, 8, None, None, saved)
    t[1, 0, 3] = float("nan")
    t[1, -1, 17] = float("inf")
    got, saved = features.group_norm(t, 8, save=True)
    ok = torch.ones(shape, dtype=torch.bool, device="cuda")
    ok[1, :, :8] = ok[1, :, 16:24] = False
    assert torch.equal(got[ok], clean[ok])
    assert torch.isnan(got[1, :, :8]).all() and torch.isnan(got[1, :, 16:24]).any()
    back, _, _ = features.group_norm_backward(dy, t, 8, None, None, saved)
    assert torch.equal(back[ok], dx[ok]) and torch.isnan(back[~ok]).all()


@pytest.mark.parametrize("shape, groups", [((300, 1, 64), 8), ((20, 30, 33), 3), ((2, 3000, 48), 4)])
def test_in_place_and_columns_of_one_table(shape, groups):
    rng = np.random.default_rng(9)
    x, dy = (_dev(rng.normal(size=shape), "bf16") for _ in range(2))
    want, saved = features.group_norm(x, groups, activation="silu", save=True)
    c = shape[-1]
    table = torch.zeros(*shape[:-1], 2 * c + 3, device="cuda", dtype=torch.bfloat16)
    table[..., 1:c + 1] = x
    view = table[..., 1:c + 1]
    side = table[..., c + 1:2 * c + 1]
    assert features.group_norm(view, groups, activation="silu", out=side) is side
    assert torch.equal(side, want) and torch.equal(view, x)
    assert torch.equal(features.group_norm(view, groups, activation="silu", out=view), want)
    with pytest.raises(_lib.NativeCallError, match="shares memory"):
        features.group_norm(view, groups, out=table[..., 2:c + 2])


def test_streams_and_graph_replays():
    rng = np.random.default_rng(10)
    sets = []
    for shape, groups in (((700, 1, 40), 5), ((9, 33, 24), 4), ((2, 5000, 40), 5)):
        sets.append((_dev(rng.normal(size=shape), "bf16"), _dev(rng.normal(size=shape), "bf16"),
                     groups, _dev(rng.normal(size=shape[-1]), "f32"),
                     _dev(rng.normal(size=shape[-1]), "f32")))

    def work():
        out = []
        for x, dy, groups, w, b in sets:
            y, saved = features.group_norm(x, groups, w, b, activation="gelu", save=True)
            out += [y, *features.group_norm_backward(dy, x, groups, w, b, saved,
                                                     activation="gelu")]
        return out

    want = work()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = work()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graphs = []
    for _ in range(2):  # two graphs, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, work()))
    for _ in range(3):
        for graph, held in graphs:
            for t in held:
                t.fill_(-1.0)
            graph.replay()
            assert all(torch.equal(a, b) for a, b in zip(want, work()))
            assert all(torch.equal(a, b) for a, b in zip(want, held))


def test_refusals():
    x = torch.zeros(6, 4, 8, device="cuda")
    for groups in (3, 0, -1, 2.0):
        with pytest.raises(ValueError, match="groups"):
            features.group_norm(x, groups)
    with pytest.raises(ValueError, match="activation"):
        features.group_norm(x, 2, activation="tanh")
    with pytest.raises(ValueError, match="samples"):
        features.group_norm(x[0, 0], 2)
    with pytest.raises(TypeError, match="does not fit"):
        features.group_norm(x, 2, torch.zeros(8, device="cuda", dtype=torch.float16))
    with pytest.raises(ValueError, match=r"shape \(8,\)"):
        features.group_norm(x, 2, None, torch.zeros(7, device="cuda"))
    with pytest.raises(ValueError, match="collapse"):
        features.group_norm(x.transpose(0, 1), 2)
    with pytest.raises(_lib.NativeCallError, match="eps"):
        features.group_norm(x, 2, eps=float("nan"))
    with pytest.raises(ValueError, match="saved"):
        features.group_norm_backward(x, x, 2, None, None, x)
    with pytest.raises(ValueError, match="dy"):
        features.group_norm_backward(x[:1], x, 2, None, None, torch.zeros(6, 2, 2, device="cuda"))
    with pytest.raises(ValueError, match="requires a gradient"):
        features.group_norm(x.clone().requires_grad_(), 2)


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("n, l, c, groups, pad", [
    # groups within lanes, of whole vectors, and that cut vectors
    (1100, 1, 8192, 64, 0), (1100, 1, 5000, 8, 0), (600, 3, 4400, 4, 1), (300, 5, 8192, 16, 0),
    (530, 2, 5005, 7, 0),
])
def test_many_samples_in_blocks_of_groups(kind, n, l, c, groups, pad):
    """More samples than workgroups of the backward pass take at a time."""
    rng = np.random.default_rng(n + l + c)
    x = rng.normal(size=(n, l, c)) * rng.uniform(0.5, 2, (n, 1, 1)) + rng.normal(size=(n, 1, c))
    x = _dev(x, kind, pad, min(pad, 1))
    w, b = _dev(1 + 0.2 * rng.normal(size=c), kind), _dev(0.3 * rng.normal(size=c), kind)
    _check(x, _dev(rng.normal(size=(n, l, c)), kind, pad), groups, w, b, ACTS[(n + c) % 4], kind)


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("n, l, c, groups", [
    # single values; groups within a vector, of lanes, of vectors, that cut vectors; in
    # stretches; in blocks
    (6000, 1, 16, 16), (6000, 1, 16, 8), (900, 1, 64, 4), (70, 6, 64, 4), (70, 6, 60, 5),
    (3, 3000, 48, 4), (40, 1, 5000, 8),
])
def test_slopes_are_of_the_values_that_were_written(kind, n, l, c, groups):
    """Values at relu's jump: x is +1 or -1 and the bias what takes weight times the
    normalised 1 (or a value beside it) to zero within a rounding, so that z is a last bit
    of either sign.  Where y is above zero the slope is 1, elsewhere 0: with dy = 1 the
    bias' gradient counts the former."""
    rng = np.random.default_rng(n + c)
    x = rng.choice([-1.0, 1.0], (n, l, c))
    single = l * c // groups == 1
    if single:
        x *= 0.0
    x = _dev(x, kind)
    w = _dev(rng.uniform(0.5, 2, c), "f32")
    if kind == "f16":  # z is a multiple of 2^-24 2^2, above float16's half smallest, 2^-25:
        w = (1024 * w).bfloat16().float()  # xhat's last bit, 2^-24, times w's, 2^2 of 2^9
    _, saved = features.group_norm(x, groups, save=True)
    # a sample's own normalised 1, of another one in every channel
    pick = torch.from_numpy(rng.integers(0, n, c)).cuda()
    mean, rstd = (saved[pick, torch.arange(c, device="cuda") // (c // groups), k] for k in (0, 1))
    at = x[pick, 0, torch.arange(c, device="cuda")].float()
    b = -((at - mean) * rstd) * w
    y, saved = features.group_norm(x, groups, w, b, activation="relu", save=True)
    _, _, db = features.group_norm_backward(torch.ones_like(x), x, groups, w, b, saved,
                                            activation="relu")
    count = (y > 0).double().sum(dim=(0, 1))
    # (a single value is its group's mean: z is the bias, 0, wherever it is)
    assert not count.any() if single else 0 < float(count.sum()) < n * l * c
    assert torch.equal(db.double(), count)  # whole numbers below 2^24: exact in fp32
