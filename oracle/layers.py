"""Float64 restatement of the learned-feature layers and of the kernel's input
gradient (test infrastructure): formulas written out, no autograd."""

from __future__ import annotations

import math

import numpy as np

_erf = np.vectorize(math.erf, otypes=[np.float64])


def layer_norm(x, w=None, b=None, eps=1e-5):
    x = np.asarray(x, np.float64)
    xc = x - x.mean(axis=1, keepdims=True)
    xh = xc / np.sqrt((xc * xc).mean(axis=1, keepdims=True) + eps)
    return xh * (1.0 if w is None else w) + (0.0 if b is None else b)


def layer_norm_backward(dy, x, w=None, eps=1e-5):
    x, dy = np.asarray(x, np.float64), np.asarray(dy, np.float64)
    xc = x - x.mean(axis=1, keepdims=True)
    rstd = 1.0 / np.sqrt((xc * xc).mean(axis=1, keepdims=True) + eps)
    xh = xc * rstd
    g = dy * (1.0 if w is None else w)
    dx = rstd * (g - g.mean(axis=1, keepdims=True) - xh * (g * xh).mean(axis=1, keepdims=True))
    return dx, (dy * xh).sum(axis=0), dy.sum(axis=0)


def activate(act, g):
    """act(g) and its derivative."""
    if act == "relu":
        return np.maximum(g, 0.0), (g > 0).astype(np.float64)
    if act == "gelu":
        cdf = 0.5 * (1.0 + _erf(g / math.sqrt(2.0)))
        return g * cdf, cdf + g * np.exp(-0.5 * g * g) / math.sqrt(2.0 * math.pi)
    s = 0.5 * (1.0 + np.tanh(0.5 * g))
    if act == "sigmoid":
        return s, s * (1.0 - s)
    return g * s, s * (1.0 + g * (1.0 - s))


def _groups(x, groups):
    """x [samples, positions, channels] with the channels as (group, channel)."""
    return x.reshape(x.shape[0], -1, groups, x.shape[-1] // groups)


def group_norm(x, groups, w=None, b=None, act=None, eps=1e-5):
    x = np.asarray(x, np.float64)
    xc = _groups(x, groups)
    xc = xc - xc.mean(axis=(1, 3), keepdims=True)
    xh = (xc / np.sqrt((xc * xc).mean(axis=(1, 3), keepdims=True) + eps)).reshape(x.shape)
    z = xh * (1.0 if w is None else w) + (0.0 if b is None else b)
    return z if act is None else activate(act, z)[0]


def group_norm_backward(dy, x, groups, w=None, b=None, act=None, eps=1e-5):
    x, dy = np.asarray(x, np.float64), np.asarray(dy, np.float64)
    xc = _groups(x, groups)
    xc = xc - xc.mean(axis=(1, 3), keepdims=True)
    rstd = 1.0 / np.sqrt((xc * xc).mean(axis=(1, 3), keepdims=True) + eps)
    xh = (xc * rstd).reshape(x.shape)
    one = 1.0 if w is None else w
    dz = dy if act is None else dy * activate(act, xh * one + (0.0 if b is None else b))[1]
    g, h = _groups(dz * one, groups), _groups(xh, groups)
    dx = rstd * (g - g.mean(axis=(1, 3), keepdims=True)
                 - h * (g * h).mean(axis=(1, 3), keepdims=True))
    axes = tuple(range(x.ndim - 1))
    return dx.reshape(x.shape), (dz * xh).sum(axis=axes), dz.sum(axis=axes)


def gated_layer(x, wg, wu, bg=None, bu=None, act="silu"):
    g = x @ wg.T + (0.0 if bg is None else bg)
    u = x @ wu.T + (0.0 if bu is None else bu)
    return activate(act, g)[0] * u


def gated_layer_backward(dh, x, wg, wu, bg=None, bu=None, act="silu"):
    g = x @ wg.T + (0.0 if bg is None else bg)
    u = x @ wu.T + (0.0 if bu is None else bu)
    a, slope = activate(act, g)
    dg, du = dh * u * slope, dh * a
    return dg @ wg + du @ wu, dg.T @ x, du.T @ x, dg.sum(axis=0), du.sum(axis=0)


def int8_rows(x):
    """(codes, scales) of rows: 127 over the largest value, both quotients rounded to
    float32 and the products to whole numbers, ties to even."""
    x = np.asarray(x, np.float64)
    most = np.abs(x).max(axis=1)
    some = most >= 2.0 ** -120
    by = np.where(some, 127 / np.where(some, most, 1), 0).astype(np.float32).astype(np.float64)
    scale = np.where(some, most / 127, 0).astype(np.float32).astype(np.float64)
    return np.rint(x * by[:, None]).astype(np.int64), scale


def int8_layer(x, wg, bg=None, wu=None, bu=None, act=None):
    """(result, the size of its sums before they meet anything that cancels)"""
    q, s = int8_rows(x)

    def project(w, b):
        c, sw = int8_rows(w)
        p = (q.astype(np.float64) @ c.T.astype(np.float64)) * s[:, None] * sw  # (sums exact)
        return p + (0.0 if b is None else b), np.abs(p)

    y, size = project(wg, bg)
    if act is not None:
        y = activate(act, y)[0]
    if wu is not None:
        u, _ = project(wu, bu)
        y = y * u
    return y, size


def philox(counter, key):
    """The four words of Philox4x32-10 (Salmon et al. 2011) of a 128-bit counter
    and a 64-bit key, in Python integers."""
    c = [(counter >> (32 * i)) & 0xFFFFFFFF for i in range(4)]
    k = [key & 0xFFFFFFFF, (key >> 32) & 0xFFFFFFFF]
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def dropout_factor(shape, rate, seed, offset=0):
    """What every element is multiplied by: 0 or the inverse of the kept share."""
    total, cut = int(np.prod(shape)), round(rate * 65536)
    out = np.zeros(total)
    words = {}
    for e in range(total):
        q = offset + e
        if q // 8 not in words:
            words = {q // 8: philox(q // 8, seed)}
        draw = (words[q // 8][q % 8 // 2] >> (16 * (q % 2))) & 0xFFFF
        if draw >= cut:
            out[e] = 65536.0 / (65536 - cut)
    return out.reshape(shape)


def kernel(kind, ard, X, params):
    """K(X, X) in float64; kinds "rbf", "matern12", "matern32", "matern52"."""
    z = X / np.asarray(params[:-1], np.float64)
    r2 = ((z[:, None, :] - z[None, :, :]) ** 2).sum(axis=2)
    os = float(params[-1])
    if kind == "rbf":
        return os * np.exp(-0.5 * r2)
    r = np.sqrt(r2)
    if kind == "matern12":
        return os * np.exp(np.maximum(-r, -20.0) if ard else -r)
    u = r * math.sqrt({"matern32": 3.0, "matern52": 5.0}[kind])
    e = np.exp(np.maximum(-u, -20.0))
    return os * (1.0 + u + (u * u / 3.0 if kind == "matern52" else 0.0)) * e


def input_gradient(kind, ard, X, params, L, R):
    """d/dX of sum_ab K_ab (L^T R)_ab; 0 between coincident points."""
    ls = np.broadcast_to(np.asarray(params[:-1], np.float64), (X.shape[1],))
    z = X / ls
    df = z[:, None, :] - z[None, :, :]
    r2 = (df ** 2).sum(axis=2)
    r = np.sqrt(r2)
    if kind == "rbf":
        h = np.exp(-0.5 * r2)
    elif kind == "matern12":
        e = np.exp(np.maximum(-r, -20.0) if ard else -r)
        h = np.divide(e, r, out=np.zeros_like(r), where=r > 0)
    elif kind == "matern32":
        h = 3.0 * np.exp(np.maximum(-math.sqrt(3.0) * r, -20.0))
    else:
        u = math.sqrt(5.0) * r
        h = 5.0 / 3.0 * (1.0 + u) * np.exp(np.maximum(-u, -20.0))
    W = L.T @ R
    h = h * (W + W.T) * float(params[-1])
    return -(h[:, :, None] * df).sum(axis=1) / ls
