"""The kernel's input gradient on the device against its float64 formula.

Tolerance, on the 2-norm of the difference over that of the result: every
entry is an fp32 sum of n weighted differences whose terms carry about ten
roundings, 2^-24 (10 + sqrt(n)) of the terms' norm; the terms cancel to a
result about sqrt(n) smaller than their sum of sizes, so that ten roundings
stay ten.  TOL = 4e-6 covers n up to 2000; the terms' scale is used where the
result itself cancels."""

import numpy as np
import pytest
import torch

from mojogp_amd import RBF, RQ, _lib
from mojogp_amd._provider import NativeProvider
from oracle import layers as ol

pytestmark = pytest.mark.gpu

KINDS = ("rbf", "matern12", "matern32", "matern52")
TOL = 4e-6


def _inputs(n, d, t, ard, seed=0, spread=1.0):
    rng = np.random.default_rng([n, d, t, seed])
    X = (spread * rng.normal(size=(n, d))).astype(np.float32)
    ls = np.sqrt(d) * rng.uniform(0.6, 1.2, size=d if ard else 1)
    params = np.append(ls, 1.3).astype(np.float32)
    return X, params, *(rng.normal(size=(t, n)).astype(np.float32) for _ in range(2))


def _check(kind, ard, X, params, L, R, tol=TOL):
    want = ol.input_gradient(kind, ard, X.astype(np.float64), params, L.astype(np.float64),
                             R.astype(np.float64))
    p = NativeProvider(kind, ard, X, params, 0.1)
    try:
        host = p.input_gradient(L, R)
        dev = p.input_gradient_device(torch.from_numpy(L).cuda(), torch.from_numpy(R).cuda())
    finally:
        p.close()
    assert host.shape == X.shape and host.dtype == np.float32
    assert np.array_equal(dev.cpu().numpy(), host)
    assert np.linalg.norm(host - want) <= tol * np.linalg.norm(want) + 1e-30
    return host


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("ard", [False, True])
@pytest.mark.parametrize("n, d, t", [(2, 1, 1), (7, 2, 3), (130, 3, 11), (257, 5, 16),
                                     (500, 8, 17), (300, 16, 1), (200, 32, 33)])
def test_against_formula(kind, ard, n, d, t):
    _check(kind, ard, *_inputs(n, d, t, ard))


@pytest.mark.parametrize("d", [4, 6, 7, 10, 12, 20, 24])
def test_dimension_steps(d):
    _check("matern52", True, *_inputs(150, d, 5, True))


@pytest.mark.parametrize("kind", KINDS)
def test_one_point_and_coincident_points(kind):
    X, params, L, R = _inputs(1, 3, 2, True)
    assert not _check(kind, True, X, params, L, R).any()
    X, params, L, R = _inputs(40, 3, 2, True)
    X[7:20] = X[6]
    _check(kind, True, X, params, L, R)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("ard", [False, True])
def test_far_points(kind, ard):
    """Points hundreds of lengthscales apart: clamped exponentials, and near
    pairs inside far clusters, whose differences keep their digits."""
    X, params, L, R = _inputs(120, 2, 3, ard, spread=400.0)
    X[60:] = X[:60] + np.float32(0.25) * np.sign(X[:60])
    # the scaled coordinates are rounded: 2^-24 of 1000 lengthscales against
    # differences of 0.2
    _check(kind, ard, X, params, L, R, tol=2.0 ** -24 * 1000 / 0.2 * 4)


def test_many_points_split_and_repeat():
    """More than one split of the columns; every call gives the same bits."""
    X, params, L, R = _inputs(2000, 4, 11, True)
    p = NativeProvider("matern52", True, X, params, 0.1)
    try:
        a = p.input_gradient(L, R)
        assert np.array_equal(a, p.input_gradient(L, R))
        p.update_params(params * np.float32(1.5))
        b = p.input_gradient(L, R)
    finally:
        p.close()
    for got, prm in ((a, params), (b, params * np.float32(1.5))):
        want = ol.input_gradient("matern52", True, X.astype(np.float64), prm,
                                 L.astype(np.float64), R.astype(np.float64))
        assert np.linalg.norm(got - want) <= TOL * np.linalg.norm(want)


def test_against_differences_of_the_product():
    """d/dt of L^T K(X + t V) R through the provider's own forward product."""
    X, params, L, R = _inputs(300, 3, 4, True, seed=1)
    V = np.random.default_rng(2).normal(size=X.shape).astype(np.float32)
    step = np.float32(1e-2)
    values = []
    for s in (1, -1):
        p = NativeProvider("rbf", True, X + s * step * V, params, 0.0)
        values.append(float((L.astype(np.float64) * p.forward_matvec(R)).sum()))
        p.close()
    p = NativeProvider("rbf", True, X, params, 0.0)
    g = p.input_gradient(L, R)
    p.close()
    got = float((g.astype(np.float64) * V).sum())
    # truncation step^2 / 6 of third derivatives of order one, products good to 2e-6 of |L| |K R|
    scale = np.linalg.norm(g) * np.linalg.norm(V)
    assert abs(got - (values[0] - values[1]) / (2 * float(step))) <= 1e-3 * scale


def test_device_call_follows_the_current_stream():
    X, params, L, R = _inputs(400, 4, 3, False)
    p = NativeProvider("rbf", False, X, params, 0.1)
    side = torch.cuda.Stream()
    try:
        want = p.input_gradient(L, R)
        with torch.cuda.stream(side):  # the inputs are still being made on it
            l, r = (torch.from_numpy(a).cuda(non_blocking=True) * 2.0 for a in (L, R))
            got = p.input_gradient_device(l * 0.5, r * 0.5)
        assert np.array_equal(got.cpu().numpy(), want)
        out = torch.empty_like(got)
        assert p.input_gradient_device(torch.from_numpy(L).cuda(), torch.from_numpy(R).cuda(),
                                       out=out) is out
        assert np.array_equal(out.cpu().numpy(), want)
        one = p.input_gradient_device(torch.from_numpy(L[0]).cuda(), torch.from_numpy(R[0]).cuda())
        assert np.array_equal(one.cpu().numpy(), p.input_gradient(L[0], R[0]))
    finally:
        p.close()


def test_refusals():
    X, params, L, R = _inputs(30, 2, 3, False)
    p = NativeProvider("rbf", False, X, params, 0.1)
    l, r = torch.from_numpy(L).cuda(), torch.from_numpy(R).cuda()
    try:
        with pytest.raises(ValueError, match="same shape"):
            p.input_gradient(L, R[:2])
        with pytest.raises(ValueError, match="shape"):
            p.input_gradient_device(l, r[:2])
        with pytest.raises(ValueError, match="float32"):
            p.input_gradient_device(l.half(), r.half())
        with pytest.raises(ValueError, match="device tensor"):
            p.input_gradient_device(l.cpu(), r.cpu())
        with pytest.raises(ValueError, match="contiguous"):
            p.input_gradient_device(torch.zeros(3, 60, device="cuda")[:, :30], r)
        with pytest.raises(ValueError, match="Lf"):
            p.input_gradient_device(l[:0], r[:0])
        with pytest.raises(_lib.NativeCallError, match="bad arguments"):
            _lib.call("mgp_input_gradient", p.handle, _lib.fptr(L), _lib.fptr(R), 0,
                      _lib.fptr(X))
    finally:
        p.close()
    tree = NativeProvider(None, False, X, np.linspace(0.9, 1.3, 5).astype(np.float32), 0.1,
                          tree_spec=(RBF() + RQ()).to_tree_spec(2))
    try:
        with pytest.raises(_lib.NativeCallError, match="kernel trees"):
            tree.input_gradient(L, R)
    finally:
        tree.close()


def _reference(kind, X, params, L, R):
    """ol.input_gradient a block of rows at a time, for thousands of points."""
    X, L, R = (a.astype(np.float64) for a in (X, L, R))
    ls = np.broadcast_to(params[:-1].astype(np.float64), (X.shape[1],))
    z, out = X / ls, np.empty_like(X)
    for i in range(0, X.shape[0], 500):
        df = z[i:i + 500, None, :] - z[None, :, :]
        r2 = np.einsum("abq,abq->ab", df, df)
        u = np.sqrt({"rbf": 1.0, "matern32": 3.0, "matern52": 5.0}[kind] * r2)
        h = {"rbf": lambda: np.exp(-0.5 * r2), "matern32": lambda: 3.0 * np.exp(-u),
             "matern52": lambda: 5.0 / 3.0 * (1.0 + u) * np.exp(-u)}[kind]()
        h *= L[:, i:i + 500].T @ R + R[:, i:i + 500].T @ L
        out[i:i + 500] = -params[-1] / ls * np.einsum("ab,abq->aq", h, df)
    return out


@pytest.mark.parametrize("kind", ["rbf", "matern32", "matern52"])
@pytest.mark.parametrize("n, d, t", [(4000, 8, 11), (4001, 1, 1), (4111, 9, 16), (4500, 16, 20),
                                     (4015, 19, 5), (4100, 24, 3), (4097, 30, 6)])
def test_matrix_core_route(kind, n, d, t):
    """Sets large enough for the matrix cores, over operand counts and ragged
    ends; two levels of fp32 sums: the tolerance of the smaller sets holds."""
    X, params, L, R = _inputs(n, d, t, True, seed=3)
    params[:-1] *= np.float32(1.5)  # norms below the route's bounds
    want = _reference(kind, X, params, L, R)
    p = NativeProvider(kind, True, X, params, 0.1)
    try:
        got = p.input_gradient(L, R)
        assert np.array_equal(got, p.input_gradient(L, R))
    finally:
        p.close()
    assert np.linalg.norm(got - want) <= TOL * np.linalg.norm(want)


def test_routes_agree_across_the_norm_bound():
    """The same points and lengthscales, once beside an outlier whose norm sends
    them to the differences: its own weight is zero, so nothing else changes."""
    X, params, L, R = _inputs(4200, 5, 7, True, seed=4)
    far = np.vstack([X, np.full((1, 5), 60.0, np.float32)])
    zero = np.zeros((7, 1), np.float32)
    a, b = NativeProvider("matern52", True, X, params, 0.1), \
        NativeProvider("matern52", True, far, params, 0.1)
    try:
        ga = a.input_gradient(L, R)
        gb = b.input_gradient(np.hstack([L, zero]), np.hstack([R, zero]))
    finally:
        a.close()
        b.close()
    assert not np.array_equal(ga, gb[:-1]) and not gb[-1].any()
    assert np.linalg.norm(ga - gb[:-1]) <= TOL * np.linalg.norm(ga)


def test_calls_in_flight_are_waited_for():
    """Calls of one handle on two streams share its work buffers, parameters
    change and the handle goes while a call may still run: every result is
    that of the parameters at its call."""
    X, params, L, R = _inputs(6000, 4, 11, True, seed=5)
    p = NativeProvider("rbf", True, X, params, 0.1)
    l, r = torch.from_numpy(L).cuda(), torch.from_numpy(R).cuda()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    first = p.input_gradient(L, R)
    got = []
    for k in range(6):
        with torch.cuda.stream(streams[k % 2]):
            got.append(p.input_gradient_device(l, r))
    p.update_params(params * np.float32(1.3))
    with torch.cuda.stream(streams[0]):
        late = p.input_gradient_device(l[:3], r[:3])
    p.close()
    torch.cuda.synchronize()
    assert all(np.array_equal(g.cpu().numpy(), first) for g in got)
    q = NativeProvider("rbf", True, X, params * np.float32(1.3), 0.1)
    try:
        assert np.array_equal(late.cpu().numpy(), q.input_gradient(L[:3], R[:3]))
    finally:
        q.close()
