"""The layers in 8-bit integers on the device against their float64 formulas.

Codes, scales and sums are exact.  What follows rounds in fp32: the sum's
conversion, its product with the row's scale, and the fused product with the channel's
and the bias (3 * 2^-24 of the sum's size, 2^-24 of the result), the activation
(4e-6 relative to the norm, as the gated layer's) and the result's own rounding."""

import numpy as np
import pytest
import torch

from mojogp_amd import _lib, features
from oracle import layers as ol

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
UNIT = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
U, F32 = 2.0 ** -24, 4e-6


def _dev(a, kind, pad=0, shift=0):
    """Rounded to `kind` on the device, in rows of a wider table of NaN."""
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


# rows x width -> hidden: both few-row kernels, both tiles, sizes that fit neither
SHAPES = [(1, 1, 1), (1, 512, 96), (3, 7, 5), (16, 33, 17), (16, 4100, 40), (17, 64, 40),
          (32, 100, 33), (33, 130, 64), (64, 1000, 24), (130, 64, 128), (129, 257, 131),
          (500, 256, 1030), (700, 17, 600), (2000, 391, 515), (8192, 256, 1024), (4000, 128, 4100),
          (300, 5000, 130), (9000, 16, 40)]


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("rows, width, hidden", SHAPES)
def test_layer(kind, rows, width, hidden):
    rng = np.random.default_rng(rows + 7 * width + 31 * hidden)
    pad = (0, 5, 8)[(rows + hidden) % 3]
    x = rng.normal(size=(rows, width)) * np.exp(rng.normal(size=(rows, 1)))
    x[rows // 2] = 0.0
    x = _dev(x, kind, pad, min(pad, 1))
    w, b = _dev(rng.normal(size=(hidden, width)), kind, pad), _dev(rng.normal(size=hidden), kind)
    q = features.int8_weights(w)
    code, scale = ol.int8_rows(_host(w))
    assert np.array_equal(q.codes[:, :width].cpu().numpy(), code)
    assert not q.codes[:, width:].any() and q.codes.shape[1] == -(-width // 16) * 16
    assert np.array_equal(_host(q.scale), scale)
    for bias in (b, None):
        y = features.int8_layer(x, q, bias)
        want, size = ol.int8_layer(_host(x), _host(w), None if bias is None else _host(b))
        assert y.dtype == TYPES[kind] and tuple(y.shape) == want.shape
        tol = 4 * U * size + (U + (UNIT[kind] if kind != "f32" else 0)) * 1.01 * np.abs(want) \
            + (2.0 ** -25 if kind == "f16" else 0)  # half a step of f16's smallest
        most = 65504.0 if kind == "f16" else np.inf
        ok = np.abs(want) < most
        assert (np.abs(_host(y) - want)[ok] <= tol[ok]).all()


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("act", sorted(features.ACTIVATIONS))
@pytest.mark.parametrize("rows, width, hidden", [(5, 40, 50), (40, 72, 88), (900, 200, 333),
                                                 (5000, 130, 700)])
def test_gated_layer(kind, act, rows, width, hidden):
    rng = np.random.default_rng(rows)
    x = _dev(rng.normal(size=(rows, width)), kind, 3)
    wg, wu = (_dev(rng.normal(size=(hidden, width)) / np.sqrt(width), kind) for _ in range(2))
    bg, bu = (_dev(0.3 * rng.normal(size=hidden), kind) for _ in range(2))
    qg, qu = features.int8_weights(wg), features.int8_weights(wu)
    for biases in ((bg, bu), (None, bu), (None, None)):
        y = features.int8_gated_layer(x, qg, qu, *biases, activation=act)
        b = [None if t is None else _host(t) for t in biases]
        want, _ = ol.int8_layer(_host(x), _host(wg), b[0], _host(wu), b[1], act)
        assert np.linalg.norm(_host(y) - want) <= (UNIT[kind] + F32) * np.linalg.norm(want)
    y = features.int8_layer(x, qg, bg, activation=act)
    want, _ = ol.int8_layer(_host(x), _host(wg), _host(bg), act=act)
    assert np.linalg.norm(_host(y) - want) <= (UNIT[kind] + F32) * np.linalg.norm(want)


@pytest.mark.parametrize("kind", sorted(TYPES))
def test_near_the_layer_itself(kind):
    """Against the gated layer in its own type: each side of a product is rounded by
    up to 1 / 254 of its row's largest value, about 3.2 of the spread for 256 values,
    uniformly: 3.2 / 127 / sqrt(12) = 0.7 % of its norm a side, in each of the
    projections: below 2 % of the result with both, and the activation's slope."""
    rng = np.random.default_rng(1)
    x = _dev(rng.normal(size=(700, 256)), kind)
    w = [_dev(rng.normal(size=(300, 256)) / 16, kind) for _ in range(2)]
    want = features.gated_layer(x, *w).double()
    got = features.int8_gated_layer(x, *map(features.int8_weights, w)).double()
    assert float((got - want).norm()) <= 0.03 * float(want.norm())


@pytest.mark.parametrize("rows", [4, 40, 600])
def test_rows_are_their_own(rows):
    """A row's result is the same beside any others; rows that are not finite, and
    no others, are NaN; tiny ones are zeros."""
    rng = np.random.default_rng(rows)
    x = _dev(rng.normal(size=(rows, 100)), "f32")
    w, b = features.int8_weights(_dev(rng.normal(size=(200, 100)), "f32")), _dev(
        rng.normal(size=200), "f32")
    clean = features.int8_layer(x, w, b)
    for r in (0, rows - 1):
        one = features.int8_layer(x[r], w, b)
        assert one.shape == (200,) and torch.equal(one, clean[r])
    x[0, 99], x[1, 0] = float("inf"), float("nan")
    x[2] *= 1e-38
    got = features.int8_layer(x, w, b)
    assert torch.isnan(got[:2]).all() and torch.equal(got[2], b)
    assert torch.equal(got[3:], clean[3:])
    broken = _dev(rng.normal(size=(200, 100)), "f32")
    broken[7, 3] = float("inf")
    got = features.int8_layer(x[3:], features.int8_weights(broken), b)
    assert torch.isnan(got[:, 7]).all() and not torch.isnan(got[:, :7]).any()


def test_sums_at_their_largest():
    """All codes at 127 over the widest rows: the sums pass 2^30."""
    x, w = torch.ones(20, 131072, device="cuda"), torch.ones(20, 131072, device="cuda")
    x[1::2] *= -1
    q = features.int8_weights(w)
    for rows in (3, 20):
        y = _host(features.int8_layer(x[:rows], q))
        want = 131072 * 127 ** 2 * float(q.scale[0].double()) ** 2
        assert (np.abs(np.abs(y) - want) <= 4 * U * want).all() and (y[1::2] < 0).all()


def test_shapes_and_empty():
    rng = np.random.default_rng(5)
    x = torch.from_numpy(rng.normal(size=(3, 4, 5, 24))).float().cuda()
    w = features.int8_weights(_dev(rng.normal(size=(32, 24)), "f32"))
    y = features.int8_layer(x, w)
    assert torch.equal(y.view(-1, 32), features.int8_layer(x.view(-1, 24), w))
    assert features.int8_layer(x[:0], w).shape == (0, 4, 5, 32)
    assert features.int8_gated_layer(x[:, :0], w, w).shape == (3, 0, 5, 32)
    table = torch.zeros(60, 70, device="cuda")
    out = table[:, 3:35]
    assert features.int8_layer(x.view(-1, 24), w, out=out) is out
    assert torch.equal(out, y.view(-1, 32)) and not table[:, :3].any() and not table[:, 35:].any()
    half = features.Int8Weights(w.codes[8:24], w.scale[8:24], 24)  # some of the channels
    assert torch.equal(features.int8_layer(x, half), y[..., 8:24])


def test_streams_and_graph_replays():
    rng = np.random.default_rng(6)
    x = {n: _dev(rng.normal(size=(n, 200)), "bf16") for n in (2, 40, 3000)}
    w = [features.int8_weights(_dev(rng.normal(size=(130, 200)), "bf16")) for _ in range(2)]

    def work():
        return [t for v in x.values() for t in (features.int8_layer(v, w[0]),
                                                features.int8_gated_layer(v, *w))]

    want = work()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = work()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = work()
    for _ in range(3):
        for t in held:
            t.fill_(-1.0)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(want, work()))
        assert all(torch.equal(a, b) for a, b in zip(want, held))


def test_refusals():
    x = torch.zeros(6, 24, device="cuda")
    w = features.int8_weights(torch.zeros(5, 24, device="cuda"))
    other = features.int8_weights(torch.zeros(4, 24, device="cuda"))
    wide = features.int8_weights(torch.zeros(5, 30, device="cuda"))
    for call, err, what in (
            (lambda: features.int8_layer(x, x), TypeError, "int8_weights"),
            (lambda: features.int8_layer(x, wide), ValueError, "24 columns"),
            (lambda: features.int8_layer(x, w._replace(codes=w.codes[:, :24])), ValueError, "codes"),
            (lambda: features.int8_layer(x, w._replace(scale=w.scale[:4])), ValueError, "scale"),
            (lambda: features.int8_layer(x, w, x[0]), ValueError, "bias"),
            (lambda: features.int8_layer(x, w, activation="tanh"), ValueError, "activation"),
            (lambda: features.int8_gated_layer(x, w, other), ValueError, "w_up"),
            (lambda: features.int8_gated_layer(x, w, w, activation=None), ValueError, "activation"),
            (lambda: features.int8_layer(x.double(), w), TypeError, "float32"),
            (lambda: features.int8_layer(x.T, w), ValueError, "unit stride"),
            (lambda: features.int8_layer(x, w, out=x[:, :4]), ValueError, "out"),
            (lambda: features.int8_layer(x, w, out=x[:, :5]), _lib.NativeCallError, "shares"),
            (lambda: features.int8_weights(x[0]), ValueError, "w must"),
            (lambda: features.int8_weights(torch.zeros(1, 131073, device="cuda")),
             _lib.NativeCallError, "131072"),
            (lambda: features.int8_layer(x.clone().requires_grad_(), w), ValueError, "gradient")):
        with pytest.raises(err, match=what):
            call()


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("rows, width, hidden", [(1, 2453, 17), (1, 2470, 17), (4, 1500, 4097),
                                                 (16, 614, 40), (16, 615, 40), (7, 4001, 33),
                                                 (5, 700, 9001), (16, 130, 8200)])
def test_few_wide_rows(kind, rows, width, hidden):
    """Up to 16 rows in one launch, with codes of their own before it, and in tiles."""
    rng = np.random.default_rng(width)
    x = _dev(rng.normal(size=(rows, width)), kind, 1)
    wg, wu = (_dev(rng.normal(size=(hidden, width)) / np.sqrt(width), kind) for _ in range(2))
    b = _dev(0.3 * rng.normal(size=hidden), kind)
    qg, qu = features.int8_weights(wg), features.int8_weights(wu)
    for up, act in ((None, None), (qu, "silu")):
        if up is None:
            y = features.int8_layer(x, qg, b)
            want, _ = ol.int8_layer(_host(x), _host(wg), _host(b))
        else:
            y = features.int8_gated_layer(x, qg, up, b, activation=act)
            want, _ = ol.int8_layer(_host(x), _host(wg), _host(b), _host(wu), None, act)
        assert np.linalg.norm(_host(y) - want) <= (UNIT[kind] + F32) * np.linalg.norm(want)
