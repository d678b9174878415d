"""The dense feed-forward operators in 64 bits, and how far a result computed
in f32 with one rounding to bf16 may be from them.

Bounds, each counted from what the kernels do:
  sums       K products of bf16 values (exact in f32) added in f32 in some
             order: at most (K + 8) * 2^-24 * sum |x w| (+ |b|).
  act        its slope is at most 1.13 and its second derivative at most 1.1 (gelu), so an
             error of the sum passes with these factors; evaluated from a
             hardware exp2 / reciprocal or erf good to a few 2^-23 relative, of
             an argument of up to 2|v|: 2^-20 |z| (1 + min(|z|^3, 64)).
  clamp, relu  where the sum is within its error of the corner, the slope may
             be either side's: the whole value is allowed.
  rounding   half a step of bf16, 2^-8 of the value.
"""
import math

import numpy as np

NONE, RELU, SILU, GELU, GELU_TANH = range(5)
ACTS = [NONE, RELU, SILU, GELU, GELU_TANH]
HALF = 2.0 ** -8
_erf = np.vectorize(math.erf, otypes=[np.float64])


def sigmoid(z):
    with np.errstate(over="ignore"):
        return np.where(z >= 0, 1 / (1 + np.exp(-np.abs(z))), np.exp(-np.abs(z)) / (1 + np.exp(-np.abs(z))))


def _phi(z):
    return 0.5 * (1 + _erf(z / math.sqrt(2)))


_C, _A = math.sqrt(2 / math.pi), 0.044715


def act(a, z):
    if a == RELU:
        return np.where(z < 0, 0.0, z)
    if a == SILU:
        return z * sigmoid(z)
    if a == GELU:
        return z * _phi(z)
    if a == GELU_TANH:
        return z * sigmoid(2 * _C * (z + _A * z ** 3))
    return z


def slope(a, z):
    if a == RELU:
        return (z > 0).astype(np.float64)
    if a == SILU:
        s = sigmoid(z)
        return s * (1 + z * (1 - s))
    if a == GELU:
        return _phi(z) + z * np.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if a == GELU_TANH:
        s = sigmoid(2 * _C * (z + _A * z ** 3))
        return s + z * s * (1 - s) * 2 * _C * (1 + 3 * _A * z * z)
    return np.ones_like(z)


def _eval(z):
    """The activation's (and its slope's) own error at z."""
    return 2.0 ** -20 * (np.abs(z) + 2.0 ** -10) * (1 + np.minimum(np.abs(z) ** 3, 64.0))


def product(x, w):
    """x w^T and the bound of its error in f32."""
    return x @ w.T, (x.shape[1] + 8) * 2.0 ** -24 * (np.abs(x) @ np.abs(w).T)


def linear(x, w, bias, residual, a):
    z, e = product(x, w)
    if bias is not None:
        z, e = z + bias, e + 2.0 ** -23 * (np.abs(z) + np.abs(bias))
    y = act(a, z)
    tol = e if a == NONE else 1.13 * e + _eval(z)
    if residual is not None:
        y = y + residual
        tol = tol + 2.0 ** -23 * (np.abs(y) + np.abs(residual))
    return y, tol + HALF * np.abs(y) + 1e-38


def gated(x, wg, wu, a, limit):
    lim = limit or math.inf
    g, eg = product(x, wg)
    u, eu = product(x, wu)
    gc, uc = np.minimum(g, lim), np.clip(u, -lim, lim)
    h = act(a, gc) * uc
    tol = np.abs(uc) * (1.13 * eg + _eval(gc)) + (np.abs(act(a, gc)) + 1.13 * eg) * eu
    return h, tol + HALF * np.abs(h) + 1e-38


def dz_linear(x, w, bias, dy, a):
    """[(dz, bound)], dz rounded to bf16."""
    z, e = product(x, w)
    if bias is not None:
        z, e = z + bias, e + 2.0 ** -23 * (np.abs(z) + np.abs(bias))
    dz = dy * slope(a, z)
    ez = np.abs(dy) * ((np.abs(z) <= e) if a == RELU else 1.1 * e + _eval(z)) + HALF * np.abs(dz)
    return [(dz, ez)]


def linear_backward(x, w, bias, dy, a):
    """{dx, dw, db}: (value, bound)."""
    [(dz, ez)] = [(dy, np.zeros_like(dy))] if a == NONE else dz_linear(x, w, bias, dy, a)
    return _grads(x, [(w, dz, ez)])


def dz_gated(x, wg, wu, dh, a, limit):
    """[(dg, bound), (du, bound)], both rounded to bf16."""
    lim = limit or math.inf
    g, eg = product(x, wg)
    u, eu = product(x, wu)
    gc, uc = np.minimum(g, lim), np.clip(u, -lim, lim)
    s, v = slope(a, gc), act(a, gc)
    dg = np.where(g > lim, 0.0, dh * uc * s)
    du = np.where(np.abs(u) > lim, 0.0, dh * v)
    es = (np.abs(g) <= eg).astype(np.float64) if a == RELU else 1.1 * eg + _eval(gc)
    near = np.abs(g - lim) <= eg
    tg = np.abs(dh) * ((np.abs(s) + es) * eu + np.abs(uc) * es) + near * np.abs(dh * uc * s) + HALF * np.abs(dg)
    near = np.abs(np.abs(u) - lim) <= eu
    tu = np.abs(dh) * (1.13 * eg + _eval(gc)) + near * np.abs(dh * v) + HALF * np.abs(du)
    return [(dg, tg), (du, tu)]


def gated_backward(x, wg, wu, dh, a, limit):
    (dg, tg), (du, tu) = dz_gated(x, wg, wu, dh, a, limit)
    return _grads(x, [(wg, dg, tg), (wu, du, tu)])


def _grads(x, parts):
    M, N = parts[0][1].shape
    dx, tx, out = 0.0, 0.0, {}
    for i, (w, dz, ez) in enumerate(parts):
        dx = dx + dz @ w
        tx = tx + ez @ np.abs(w) + (len(parts) * N + 8) * 2.0 ** -24 * (np.abs(dz) @ np.abs(w))
        dw = dz.T @ x
        tw = ez.T @ np.abs(x) + (M + 8) * 2.0 ** -24 * (np.abs(dz).T @ np.abs(x))
        out["dw%d" % i] = (dw, tw + HALF * np.abs(dw) + 1e-38)
    out["dx"] = (dx, tx + HALF * np.abs(dx) + 1e-38)
    db, dz, ez = parts[0][1].sum(0), parts[0][1], parts[0][2]
    out["db"] = (db, ez.sum(0) + (M + 8) * 2.0 ** -24 * np.abs(dz).sum(0) + HALF * np.abs(db) + 1e-38)
    return out


def check(got, want, tol, what, rms=HALF):
    """got: f64 values of bf16 codes. Every element within its bound, and (the
    bounds of long sums being the worst case) the whole within `rms` of the
    2-norm: the rms of a rounding is at most 2^-8 / sqrt(3), of two (an operand's
    and the output's) 2^-8 * 0.82."""
    assert got.shape == want.shape
    assert np.all(np.isfinite(got)), "%s: not finite" % what
    d = np.abs(got - want)
    i = np.unravel_index(np.argmax(d - tol), d.shape)
    assert d[i] <= tol[i], "%s: %s is %.6g, %.6g wanted, off %.3g of %.3g" % (what, i, got[i], want[i], d[i], tol[i])
    n = np.linalg.norm(want)
    if want.size >= 256:
        assert np.linalg.norm(d) <= rms * n, "%s: rms %.3g" % (what, np.linalg.norm(d) / n)
