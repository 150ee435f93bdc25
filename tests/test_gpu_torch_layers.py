"""The learned-feature layers on the device against their float64 formulas.

Tolerances, on the 2-norm of the difference over that of the result: an output
rounded once to a type of unit roundoff u is at most u off; the fp32 sums of
up to n terms of either sign add about 2^-24 sqrt(n) (n up to 2000 rows or
columns here), taken as F32 = 4e-6.  The gated layer's gradients also carry
the rounding of dg and du, which the matrix cores take in the element type:
another u, and 2 u where both meet in dx.

(The test_gpu_torch_* modules run torch on the device; their names put them
after test_gpu_scratch_limit, which needs the free memory that the runtime
reports to be all it has: the runtime also has what it holds as scratch for
earlier kernels.)"""

import numpy as np
import pytest
import torch

from mojogp_amd import _lib, features
from oracle import layers as ol

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
UNIT = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
F32 = 4e-6


def _dev(a, kind, pad=0, shift=0):
    """The array rounded to `kind` on the device, in rows of a wider table
    (`pad` more columns, the first `shift` skipped); NaN around it."""
    a = np.asarray(a, np.float64)
    if a.ndim == 1:
        return torch.from_numpy(a).to("cuda", TYPES[kind])
    wide = torch.full((a.shape[0], a.shape[1] + pad), float("nan"), dtype=TYPES[kind],
                      device="cuda")
    view = wide[:, shift:shift + a.shape[1]]
    view.copy_(torch.from_numpy(a))
    return view


def _host(t):
    return t.double().cpu().numpy()


def _check(got, want, tol, dtype=None):
    assert tuple(got.shape) == want.shape
    if dtype is not None:
        assert got.dtype == dtype
    err = np.linalg.norm(_host(got) - want)
    assert err <= tol * np.linalg.norm(want) + 1e-30, (err, np.linalg.norm(want))


# ---------------------------------------------------------------- layer norm

NORM = [(1, 1, 0), (3, 8, 0), (5, 7, 0), (17, 33, 5), (64, 256, 0), (33, 771, 13), (2, 1024, 0),
        (1500, 1100, 0), (1030, 2048, 8), (2, 4096, 0), (3, 8191, 0), (2, 8192, 0), (3, 8193, 0),
        (70, 20001, 3), (1100, 16, 0), (300, 130, 0), (1300, 513, 0)]


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("rows, width, pad", NORM)
def test_layer_norm(kind, rows, width, pad):
    rng = np.random.default_rng(rows * 31 + width)
    x = _dev(rng.normal(size=(rows, width)) * rng.uniform(0.5, 2, (rows, 1))
             + rng.normal(size=(rows, 1)), kind, pad)
    w, b = _dev(1 + 0.1 * rng.normal(size=width), kind), _dev(rng.normal(size=width), kind)
    dy = _dev(rng.normal(size=(rows, width)), kind, pad, min(pad, 1))
    y, saved = features.layer_norm(x, w, b, save=True)
    dx, dw, db = features.layer_norm_backward(dy, x, w, saved)
    X, W, DY = _host(x), _host(w), _host(dy)
    tol = UNIT[kind] + F32
    _check(y, ol.layer_norm(X, W, _host(b)), tol, TYPES[kind])
    rdx, rdw, rdb = ol.layer_norm_backward(DY, X, W)
    if width > 1:  # the gradients of a single column are zero
        _check(dx, rdx, tol, TYPES[kind])
        _check(dw, rdw, tol, TYPES[kind])
    else:
        assert not dx.any() and not dw.any()
    _check(db, rdb, tol, TYPES[kind])


@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_layer_norm_float32_parameters(kind, rng):
    x, dy = _dev(rng.normal(size=(40, 72)), kind), _dev(rng.normal(size=(40, 72)), kind)
    w, b = _dev(rng.normal(size=72), "f32"), _dev(rng.normal(size=72), "f32")
    y, saved = features.layer_norm(x, w, b, save=True)
    dx, dw, db = features.layer_norm_backward(dy, x, w, saved)
    _check(y, ol.layer_norm(_host(x), _host(w), _host(b)), UNIT[kind] + F32, TYPES[kind])
    rdx, rdw, rdb = ol.layer_norm_backward(_host(dy), _host(x), _host(w))
    _check(dx, rdx, UNIT[kind] + F32, TYPES[kind])
    _check(dw, rdw, F32, torch.float32)
    _check(db, rdb, F32, torch.float32)


def test_layer_norm_without_parameters(rng):
    x, dy = _dev(rng.normal(size=(9, 50)), "f32"), _dev(rng.normal(size=(9, 50)), "f32")
    y, saved = features.layer_norm(x, save=True)
    dx, dw, db = features.layer_norm_backward(dy, x, None, saved, bias=False)
    assert dw is None and db is None
    _check(y, ol.layer_norm(_host(x)), F32)
    _check(dx, ol.layer_norm_backward(_host(dy), _host(x))[0], F32)


def test_layer_norm_special_rows():
    """Constant rows, a level far above the spread, and non-finite rows, which
    stay their own."""
    rng = np.random.default_rng(5)
    x = rng.normal(size=(8, 300)).astype(np.float32)
    x[1] = 3.25
    x[2] += 4096.0
    t = torch.from_numpy(x).cuda()
    clean = features.layer_norm(t)
    want = ol.layer_norm(x)
    assert not clean[1].any()
    # the mean's rounding: 2^-24 4096 of a spread of 1
    _check(clean[2:3], want[2:3], 4096 * 2.0 ** -23)
    t[4, 7] = float("inf")
    t[6, 299] = float("nan")
    got = features.layer_norm(t)
    ok = [0, 1, 2, 3, 5, 7]
    assert torch.equal(got[ok], clean[ok])
    assert torch.isnan(got[6]).all() and torch.isnan(got[4]).any()


def test_layer_norm_empty_and_many_dimensions(rng):
    e = torch.empty(0, 24, device="cuda")
    w = torch.ones(24, device="cuda")
    y, saved = features.layer_norm(e, w, save=True)
    dx, dw, db = features.layer_norm_backward(e, e, w, saved)
    assert y.shape == (0, 24) and dx.shape == (0, 24)
    assert not dw.any() and not db.any() and dw.shape == db.shape == (24,)
    x = torch.from_numpy(rng.normal(size=(2, 3, 5, 24))).float().cuda()
    y = features.layer_norm(x, w)
    assert torch.equal(y.view(-1, 24), features.layer_norm(x.view(-1, 24), w))
    assert torch.equal(features.layer_norm(x[0, 0, 0], w), y[0, 0, 0])
    out = torch.empty(30, 40, device="cuda")[:, :24]
    assert features.layer_norm(x.view(-1, 24), w, out=out) is out
    assert torch.equal(out, y.view(-1, 24))


# ---------------------------------------------------------------- gated layer

GATED = [(1, 1, 1), (1, 16, 24), (3, 7, 5), (2, 512, 96), (17, 33, 65), (64, 40, 64),
         (130, 64, 128), (129, 257, 131), (500, 256, 130), (300, 8, 600), (257, 96, 16),
         (1, 1027, 3), (700, 200, 333), (2000, 24, 40)]


def _gated(rng, rows, width, hidden, kind, pad=0):
    return (_dev(rng.normal(size=(rows, width)), kind, pad, min(pad, 1)),
            _dev(rng.normal(size=(hidden, width)) / np.sqrt(width), kind, pad),
            _dev(rng.normal(size=(hidden, width)) / np.sqrt(width), kind, pad),
            _dev(0.3 * rng.normal(size=hidden), kind), _dev(0.3 * rng.normal(size=hidden), kind))


def _gated_check(args, dh, act, kind, biased=True):
    args = args if biased else args[:3]
    h = features.gated_layer(*args, activation=act)
    g = features.gated_layer_backward(dh, *args, activation=act)
    host = [_host(a) for a in args]
    _check(h, ol.gated_layer(*host, act=act), UNIT[kind] + F32, TYPES[kind])
    ref = ol.gated_layer_backward(_host(dh), *host, act=act)
    for got, want, units in zip(g, ref, (3, 2, 2, 1, 1)):
        if got is not None:
            _check(got, want, units * UNIT[kind] + F32, TYPES[kind])
    assert biased or (g.db_gate is None and g.db_up is None)


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("rows, width, hidden", GATED)
def test_gated_layer(kind, rows, width, hidden):
    rng = np.random.default_rng(rows + 7 * width + 31 * hidden)
    act = ("silu", "gelu", "sigmoid")[(rows + hidden) % 3]
    args = _gated(rng, rows, width, hidden, kind)
    _gated_check(args, _dev(rng.normal(size=(rows, hidden)), kind), act, kind)


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("act", sorted(features.ACTIVATIONS))
@pytest.mark.parametrize("pad", [1, 8])
def test_gated_layer_strides(kind, act, pad):
    """Rows of wider tables (surrounded by NaN), aligned and not, no biases."""
    rng = np.random.default_rng(pad)
    args = _gated(rng, 150, 72, 88, kind, pad)
    dh = _dev(rng.normal(size=(150, 88)), kind, pad)
    _gated_check(args, dh, act, kind, biased=pad == 8)


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("width", [40, 128, 129])
def test_gated_layer_many_tiles(kind, width):
    """More large tiles than the device takes at a time, one, two and three steps
    of the reduction each: rows from every tile."""
    rng = np.random.default_rng(width)
    x, *weights = _gated(rng, 32760, width, 1279, kind)
    h = features.gated_layer(x, *weights)
    _check(h[::37], ol.gated_layer(_host(x[::37]), *[_host(w) for w in weights]),
           UNIT[kind] + F32, TYPES[kind])


def test_gated_layer_directional_differences():
    """The gradients against differences of the forward pass itself."""
    rng = np.random.default_rng(3)
    args = _gated(rng, 96, 40, 56, "f32")
    dh = _dev(rng.normal(size=(96, 56)), "f32")
    g = features.gated_layer_backward(dh, *args)
    step = 1e-2
    for k, grad in enumerate(g):
        v = torch.from_numpy(rng.normal(size=tuple(args[k].shape))).to("cuda", torch.float32)
        v /= v.norm()
        f = [(dh.double() * features.gated_layer(*args[:k], args[k] + s * step * v,
                                                 *args[k + 1:]).double()).sum()
             for s in (1.0, -1.0)]
        want = float(f[0] - f[1]) / (2 * step)
        # truncation step^2 f''' / 6 of unit directions, fp32 values of size ~ |h| over step
        assert abs(float((grad.double() * v.double()).sum()) - want) <= 2e-3 * float(grad.norm())


def test_gated_layer_chosen_gradients(rng):
    args = _gated(rng, 70, 24, 32, "bf16")
    dh = _dev(rng.normal(size=(70, 32)), "bf16")
    full = features.gated_layer_backward(dh, *args)
    data = features.gated_layer_backward(dh, *args, need_dx=False)
    fixed = features.gated_layer_backward(dh, *args, need_dw=False)
    assert data.dx is None and fixed.dw_gate is None and fixed.dw_up is None
    for name in ("dw_gate", "dw_up", "db_gate", "db_up"):
        assert torch.equal(getattr(data, name), getattr(full, name))
    assert torch.equal(fixed.dx, full.dx) and torch.equal(fixed.db_up, full.db_up)


@pytest.mark.parametrize("kind", sorted(TYPES))
def test_gated_layer_non_finite_rows_stay_their_own(kind, rng):
    args = _gated(rng, 200, 48, 72, kind)
    clean = features.gated_layer(*args)
    args[0][17, 3] = float("nan")
    args[0][130, 47] = float("inf")
    got = features.gated_layer(*args)
    bad = [17, 130]
    keep = [r for r in range(200) if r not in bad]
    assert torch.equal(got[keep], clean[keep])
    assert torch.isnan(got[17]).all() and not torch.isfinite(got[130]).all()


def test_gated_layer_no_rows(rng):
    args = list(_gated(rng, 4, 24, 16, "f32"))
    args[0] = args[0][:0]
    assert features.gated_layer(*args).shape == (0, 16)
    g = features.gated_layer_backward(torch.empty(0, 16, device="cuda"), *args)
    assert g.dx.shape == (0, 24)
    assert not any(t.any() for t in g[1:])


# ---------------------------------------------------------------- dropout

@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("rows, width, pad, offset", [
    (1, 1, 0, 0), (3, 5, 0, 0), (40, 64, 0, 16), (33, 77, 0, 0), (33, 77, 5, 8), (9, 40, 8, 3),
    (16, 32, 0, (1 << 35) + 8), (5, 31, 0, (1 << 63) + 5)])
def test_dropout(kind, rows, width, pad, offset):
    rng = np.random.default_rng(rows + width)
    seed = 0xFEDCBA9876543210 + rows
    x, r, dy = (_dev(rng.normal(size=(rows, width)), kind, pad) for _ in range(3))
    for rate in (0.0, 0.1, 0.5):
        f = ol.dropout_factor((rows, width), rate, seed, offset)
        tol = UNIT[kind] + 2.0 ** -22  # the scale, the product and the sum in fp32
        _check(features.dropout(x, rate, seed, offset=offset), _host(x) * f, tol, TYPES[kind])
        y = features.dropout(x, rate, seed, offset=offset, residual=r)
        _check(y, _host(x) * f + _host(r), tol, TYPES[kind])
        dx = features.dropout_backward(dy, rate, seed, offset=offset)
        assert np.array_equal(_host(dx) == 0, (_host(dy) * f) == 0)
        _check(dx, _host(dy) * f, tol, TYPES[kind])


def test_dropout_halves_of_a_step_and_in_place(rng):
    """Draws are numbered: two calls on halves draw what one call on the whole
    does, whichever kernel serves them; out may be an input."""
    x = _dev(rng.normal(size=(64, 50)), "f32")
    whole = features.dropout(x, 0.3, 11, offset=24)
    a = features.dropout(x[:21], 0.3, 11, offset=24)
    b = features.dropout(x[21:], 0.3, 11, offset=24 + 21 * 50)
    assert torch.equal(torch.cat([a, b]), whole)
    assert torch.equal(features.dropout(x, 0.3, 11, offset=24, out=x), whole)


def test_dropout_of_non_finite_values():
    x = torch.full((64, 64), float("inf"), device="cuda")
    x[::2] = float("nan")
    y = features.dropout(x, 0.5, 3)
    f = torch.from_numpy(ol.dropout_factor((64, 64), 0.5, 3)).cuda()
    assert not y[f == 0].any()
    assert torch.isinf(y[1::2][f[1::2] > 0]).all() and torch.isnan(y[::2][f[::2] > 0]).all()
    assert features.dropout(x[:0], 0.5, 3).shape == (0, 64)


# ---------------------------------------------------------------- streams, graphs, refusals

def _step(x, w, args, dh):
    y, saved = features.layer_norm(x, w, save=True)
    h = features.gated_layer(y, *args)
    z = features.dropout(h, 0.2, 5, residual=h)
    dd = features.dropout_backward(dh, 0.2, 5) + dh
    g = features.gated_layer_backward(dd, y, *args)
    return (z, *g, *features.layer_norm_backward(g.dx, x, w, saved))


def test_current_stream_and_graph_replays(rng):
    """On a stream of the caller's, and recorded into a graph that is replayed
    between eager work, every pass gives the eager result's bits."""
    args = _gated(rng, 300, 56, 72, "bf16")
    x, w = args[0], _dev(1 + 0.1 * rng.normal(size=56), "bf16")
    dh = _dev(rng.normal(size=(300, 72)), "bf16")
    want = _step(x, w, args[1:], dh)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _step(x, w, args[1:], dh)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = _step(x, w, args[1:], dh)
    for _ in range(3):
        for t in held:
            t.fill_(-1.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, held))
        assert all(torch.equal(a, b) for a, b in zip(want, _step(x, w, args[1:], dh)))


def test_refusals(rng):
    x = torch.zeros(6, 8, device="cuda")
    w = torch.zeros(5, 8, device="cuda")
    with pytest.raises(ValueError, match="device tensor"):
        features.layer_norm(x.cpu())
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        features.layer_norm(x.double())
    with pytest.raises(ValueError, match="unit stride"):
        features.layer_norm(x.T)
    with pytest.raises(ValueError, match="overlap"):
        features.layer_norm(x[:1].expand(6, 8))
    with pytest.raises(ValueError, match=r"shape \(8,\)"):
        features.layer_norm(x, torch.zeros(7, device="cuda"))
    with pytest.raises(TypeError, match="does not fit"):
        features.layer_norm(x, torch.zeros(8, device="cuda", dtype=torch.float16))
    with pytest.raises(_lib.NativeCallError, match="eps"):
        features.layer_norm(x, eps=-1.0)
    with pytest.raises(ValueError, match="saved"):
        features.layer_norm_backward(x, x, None, x)
    with pytest.raises(ValueError, match="collapse"):
        features.layer_norm(torch.zeros(4, 6, 8, device="cuda").transpose(0, 1))
    with pytest.raises(ValueError, match="at least one column"):
        features.layer_norm(x[:, :0])
    with pytest.raises(ValueError, match="activation"):
        features.gated_layer(x, w, w, activation="tanh")
    with pytest.raises(ValueError, match="w_gate"):
        features.gated_layer(x, w[:, :7], w)
    with pytest.raises(ValueError, match="w_up"):
        features.gated_layer(x, w, w[:4])
    with pytest.raises(TypeError, match="element type"):
        features.gated_layer(x, w, w.bfloat16())
    with pytest.raises(ValueError, match="dh"):
        features.gated_layer_backward(x, x, w, w)
    for rate in (-0.1, 1.0, 1.0 - 2.0 ** -20, float("nan")):
        with pytest.raises(_lib.NativeCallError, match="rate"):
            features.dropout(x, rate, 1)
    with pytest.raises(ValueError, match="seed"):
        features.dropout(x, 0.1, -1)
    with pytest.raises(_lib.NativeCallError, match="64 bits"):
        features.dropout(x, 0.1, 1, offset=(1 << 64) - 8)


def test_native_refusals():
    """The C entries check what they are given before any device work."""
    a = _lib.GatedLayer(0, 0, 4, 8, 4, 1 << 20, 8, 1 << 20, 8, 1 << 20, 8, None, None)
    with pytest.raises(_lib.NativeCallError, match="null device array h"):
        _lib.call("mgp_gated_layer_device", a, None, 4, None, 0, None)
    with pytest.raises(_lib.NativeCallError, match="workspace of 0 bytes"):
        _lib.call("mgp_gated_layer_backward_device", a, 1 << 20, 4, None, None, None, None, None,
                  None, 0, None)
    a.type = 7
    with pytest.raises(_lib.NativeCallError, match="element type"):
        _lib.call("mgp_gated_layer_device", a, 1 << 20, 4, None, 0, None)
    a.type, a.x_stride = 0, 7
    with pytest.raises(_lib.NativeCallError, match="row stride of x"):
        _lib.call("mgp_gated_layer_device", a, 1 << 20, 4, None, 0, None)
