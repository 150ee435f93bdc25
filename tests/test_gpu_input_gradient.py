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
