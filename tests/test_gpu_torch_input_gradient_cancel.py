"""Input gradients of sets that are large enough for the matrix cores, but whose
sums cancel or whose weights differ in size: points in clusters, weights on near
pairs, points with small weights beside points with large ones.

Tolerance, on the 2-norm: TOL as in test_gpu_torch_input_gradient for the sums, and
the rounding of the scaled coordinates themselves, 2^-24 |z|, which enters as
2^-24 sqrt(sum_i |z_i|^2 Q_i), Q_i = sum_b (W_ib h_ib)^2: the kernels work on
coordinates in float32, whatever the route."""

import numpy as np
import pytest

from mojogp_amd._provider import NativeProvider

pytestmark = pytest.mark.gpu

TOL = 4e-6
KINDS = ("rbf", "matern32", "matern52")
SCALE = {"rbf": np.sqrt(0.5 * np.log2(np.e)), "matern32": np.sqrt(3) * np.log2(np.e),
         "matern52": np.sqrt(5) * np.log2(np.e)}  # of the coordinates whose norm bounds the route
REACH = {"rbf": 32.0, "matern32": 256.0, "matern52": 512.0}


def _formula(kind, X, L, R):
    """The gradient for unit lengthscales in float64, and per row what the
    tolerances need: sqrt(|z|^2 Q) in units of the result, sqrt(sum (W h r)^2) and the
    same with the sum of the sizes of a weight's terms in place of W."""
    X, L, R = (a.astype(np.float64) for a in (X, L, R))
    z = X - X.mean(axis=0)
    out, q, own, terms = np.empty_like(X), *(np.empty(len(X)) for _ in range(3))
    for i in range(0, len(X), 512):
        df = X[i:i + 512, None, :] - X[None]
        r2 = (df ** 2).sum(axis=2)
        u = np.sqrt(r2 * {"rbf": 1.0, "matern32": 3.0, "matern52": 5.0}[kind])
        e = np.exp(np.maximum(-u, -20.0))  # clamped, as in oracle.layers.input_gradient
        h = {"rbf": lambda: np.exp(-0.5 * r2), "matern32": lambda: 3.0 * e,
             "matern52": lambda: 5.0 / 3.0 * (1.0 + u) * e}[kind]()
        sizes = abs(L[:, i:i + 512]).T @ abs(R) + abs(R[:, i:i + 512]).T @ abs(L)
        terms[i:i + 512] = ((h * sizes) ** 2 * r2).sum(axis=1)
        h *= L[:, i:i + 512].T @ R + R[:, i:i + 512].T @ L
        h[np.arange(len(h)), i + np.arange(len(h))] = 0.0
        out[i:i + 512] = -(h[:, :, None] * df).sum(axis=1)
        q[i:i + 512] = (h ** 2).sum(axis=1)
        own[i:i + 512] = (h ** 2 * r2).sum(axis=1)
    return out, np.sqrt((z ** 2).sum(axis=1) * q), np.sqrt(own), np.sqrt(terms)


def _gradient(kind, X, L, R):
    p = NativeProvider(kind, True, X, np.ones(X.shape[1] + 1, np.float32), 0.1)
    try:
        got = p.input_gradient(L, R)
        assert np.array_equal(got, p.input_gradient(L, R))
    finally:
        p.close()
    return got.astype(np.float64)


def _check(kind, X, L, R):
    got = _gradient(kind, X, L, R)
    want, coords, _, _ = _formula(kind, X, L, R)
    err = np.linalg.norm(got - want)
    assert err <= TOL * np.linalg.norm(want) + 2.0 ** -24 * np.linalg.norm(coords)


def _clusters(kind, n, d, radius, rng):
    """Eight clusters on the axes, 0.8 of the route's reach from the middle."""
    far = np.sqrt(0.8 * REACH[kind]) / SCALE[kind]
    centres = np.zeros((8, d))
    for c in range(8):
        centres[c, c // 2] = far * (1 if c % 2 else -1)
    X = centres[rng.permutation(np.arange(n) % 8)] + radius * rng.normal(size=(n, d))
    return X.astype(np.float32)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n, d, t", [(4096, 8, 5), (4300, 20, 17)])
@pytest.mark.parametrize("radius", [0.1, 0.01, 0.001])
def test_clusters(kind, n, d, t, radius):
    rng = np.random.default_rng([n, d, t])
    X = _clusters(kind, n, d, radius, rng)
    L, R = (rng.normal(size=(t, n)).astype(np.float32) for _ in range(2))
    _check(kind, X, L, R)


@pytest.mark.parametrize("kind", KINDS)
def test_clusters_in_some_rows_only(kind):
    """Half of the points are spread out: the blocks of rows differ in their route."""
    rng = np.random.default_rng(4)
    X = np.vstack([_clusters(kind, 2500, 8, 0.002, rng),
                   (rng.normal(size=(2500, 8)) / SCALE[kind]).astype(np.float32)])
    L, R = (rng.normal(size=(6, 5000)).astype(np.float32) for _ in range(2))
    _check(kind, X, L, R)
    got, (want, coords, _, _) = _gradient(kind, X, L, R), _formula(kind, X, L, R)
    for rows in (slice(0, 2500), slice(2500, 5000)):
        assert np.linalg.norm((got - want)[rows]) <= TOL * np.linalg.norm(want[rows]) \
            + 2.0 ** -24 * np.linalg.norm(coords[rows])


@pytest.mark.parametrize("kind", KINDS)
def test_weights_on_near_pairs(kind):
    """Columns that weigh single pairs of neighbours."""
    rng = np.random.default_rng(9)
    X = (rng.normal(size=(4200, 5)) * 1.5 / SCALE[kind]).astype(np.float32)
    L, R = (np.zeros((8, 4200), np.float32) for _ in range(2))
    for c, i in enumerate(rng.integers(0, 4200, 8)):
        near = np.argsort(((X - X[i]) ** 2).sum(axis=1))[1]
        L[c, i], R[c, near] = 1.0, 1.0
    _check(kind, X, L, R)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("case", ["points", "one point", "columns"])
def test_weights_of_different_sizes(kind, case):
    """Row by row: what a row has lost by its own sums on the matrix cores is at most
    6e-7 of sqrt(|z|^2 Q), three times that for a single row; a weight is a sum in
    22 bits or more of terms that may cancel."""
    rng = np.random.default_rng(10)
    n, t = 4500, 6
    X = (rng.normal(size=(n, 5)) / SCALE[kind]).astype(np.float32)
    L, R = rng.normal(size=(t, n)), rng.normal(size=(t, n))
    if case == "points":
        size = 10.0 ** rng.uniform(-6, 6, n)
        L, R = L * size, R * size
    elif case == "one point":
        X[7] += np.float32(5.0) / np.float32(SCALE[kind] * np.sqrt(5))
        L[:, 7] *= 1e9
    else:
        size = 10.0 ** rng.uniform(-6, 6, (t, 1))
        L, R = L * size, R / size
    L, R = L.astype(np.float32), R.astype(np.float32)
    got, (want, coords, own, terms) = _gradient(kind, X, L, R), _formula(kind, X, L, R)
    err = np.linalg.norm(got - want, axis=1)
    assert np.all(err <= 3 * 6e-7 * coords + 4 * TOL * own + 2.0 ** -21 * terms + 1e-37)


@pytest.mark.parametrize("kind", KINDS)
def test_points_in_order(kind):
    """Points in order on a line out to the route's bound, weights as those of a
    marginal likelihood: the roundings of neighbours are alike and do not average out.
    Block by block of 128 rows, twice what the route lets pass (RBF, whose values fall
    fastest with the distance: three times), beside the coordinates' rounding, here of
    sums S of one sign as well."""
    rng = np.random.default_rng(21)
    n = 10240
    X = np.zeros((n, 5))
    X[:, 0] = np.linspace(-0.9, 0.9, n) * np.sqrt(REACH[kind]) / SCALE[kind]
    X[:, 1] = 0.01 * np.sin(np.arange(n))
    X = X.astype(np.float32)
    alpha, probes = 10.0 * (np.sin(3.0 * X[:, 0]) + 0.1 * rng.normal(size=n)), \
        rng.normal(size=(10, n))
    L = np.vstack([-0.5 * alpha, probes / 20.0]).astype(np.float32)
    R = np.vstack([alpha, probes]).astype(np.float32)
    got, (want, coords, _, _) = _gradient(kind, X, L, R), _formula(kind, X, L, R)
    sums = np.empty(n)
    for i in range(0, n, 512):  # |z| sum_b W h
        df = (X[i:i + 512, None, :2] - X[None, :, :2]).astype(np.float64)
        u = np.sqrt((df ** 2).sum(axis=2) * {"rbf": 1.0, "matern32": 3.0, "matern52": 5.0}[kind])
        h = np.exp(-0.5 * u ** 2) if kind == "rbf" else np.exp(-u) * \
            (3.0 if kind == "matern32" else 5.0 / 3.0 * (1.0 + u))
        w = L[:, i:i + 512].astype(np.float64).T @ R + R[:, i:i + 512].astype(np.float64).T @ L
        sums[i:i + 512] = (h * w).sum(axis=1)
    sums *= np.linalg.norm(X - X.mean(axis=0), axis=1)
    blocks = [np.sqrt((a ** 2).reshape(n // 128, -1).sum(axis=1))
              for a in (got - want, want, coords, sums)]
    err, size, coords, sums = blocks
    times = 3 if kind == "rbf" else 2
    assert np.all(err <= times * 3e-6 * size + 2.0 ** -24 * (coords + sums))
