"""The norm, microscaled values and the products with them in 64 bits, and how
far a result computed in f32 with one rounding may be from them.

Bounds, each counted from what the kernels do:
  sums       K products added in f32 in some order: at most (K + 8) * 2^-24 *
             sum |x w|. Where one operand is MXFP8 the matrix instruction drops
             what lies more than 13 bits below the leading bit of the largest of a
             block's 32 products: 2^-13 of that product, for each of them (448 *
             1 + 0.140625 * 1 comes out as 448.125, 448 + 0.28125 exactly).
  norm       the sum of D squares is off by (D + 8) * 2^-24 relative, rstd by
             half of that and 4 roundings, y by two products more.
  rounding   half a step: 2^-8 of a bf16 value, 2^-4 of an E4M3 one (2^-10 of
             the scale below its normal numbers), 2^-2 of the scale at most for
             E2M1.
"""
import numpy as np

import ffn_ref as R

BF16, MXFP8, MXFP4 = range(3)
HALF = R.HALF
U = 2.0 ** -24


def _e4m3(c):
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e > 0, (8 + m) * 2.0 ** (e - 10.0), m * 2.0 ** -9)
    return np.where(c & 0x7F == 0x7F, np.nan, np.where(c & 0x80, -v, v))


E4M3 = _e4m3(np.arange(256))
E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6])
MOST = {MXFP8: 448.0, MXFP4: 6.0}


def scale_ld(K):
    return (K + 127) // 128 * 4


def numbers(type, codes):
    """Codes as stored -> one number a value."""
    if type == MXFP8:
        return codes
    return np.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[0], -1)


def stored(type, c):
    return c if type == MXFP8 else (c[:, 0::2] | c[:, 1::2] << 4)


def values(type, codes, scales):
    """[R, K] in 64 bits; scales as stored (rows of whole words)."""
    v = (E4M3 if type == MXFP8 else E2M1)[numbers(type, codes)]
    s = scales[:, :v.shape[1] // 32].astype(int)
    f = np.where(s == 255, np.nan, 2.0 ** (s - 127.0))
    return (v.reshape(v.shape[0], -1, 32) * f[..., None]).reshape(v.shape)


def quantize(type, v):
    """(codes as stored, scales as stored): each value's nearest number, found by
    search; a tie goes to the even code."""
    Rr, K = v.shape
    b = v.reshape(Rr, K // 32, 32)
    bad = ~np.isfinite(b).all(2)
    with np.errstate(invalid="ignore"):
        amax = np.where(bad, 0.0, np.abs(b).max(2))
    e = np.full(amax.shape, -127)
    for k in range(-127, 127):                      # the first that is large enough
        e = np.where(amax > MOST[type] * 2.0 ** k, k + 1, e)
    with np.errstate(invalid="ignore"):
        q = np.where(bad[..., None], 0.0, b / 2.0 ** e[..., None].astype(float))
    grid = (E4M3[:127] if type == MXFP8 else E2M1[:8])
    a = np.abs(q)
    hi = np.clip(np.searchsorted(grid, a), 0, len(grid) - 1)
    lo = np.maximum(hi - 1, 0)
    up, down = grid[hi] - a, a - grid[lo]
    c = np.where(up < down, hi, np.where(down < up, lo, np.where(hi % 2 == 0, hi, lo)))
    c = np.where(a == grid[hi], hi, c)
    c = (c | np.where(np.signbit(q), 0x80 if type == MXFP8 else 8, 0)).astype(np.uint8).reshape(Rr, K)
    scales = np.zeros((Rr, scale_ld(K)), np.uint8)
    scales[:, :K // 32] = np.where(bad, 255, e + 127)
    return stored(type, c), scales


def product(x, w, type):
    """x w^T of values in 64 bits, and the bound of the kernels' error."""
    z, e = R.product(x, w)
    if type == MXFP8:
        top = lambda a: np.abs(a).reshape(a.shape[0], -1, 32).max(2)  # noqa: E731
        e = e + 32 * 2.0 ** -13 * (top(x) @ top(w).T)
    return z, e


def linear(x, w, bias, residual, a, type):
    z, e = product(x, w, type)
    if bias is not None:
        z, e = z + bias, e + 2.0 ** -23 * (np.abs(z) + np.abs(bias))
    y = R.act(a, z)
    tol = e if a == R.NONE else 1.13 * e + R._eval(z)
    if residual is not None:
        y = y + residual
        tol = tol + 2.0 ** -23 * (np.abs(y) + np.abs(residual))
    return y, tol + HALF * np.abs(y) + 1e-38


def gated(x, wg, wu, a, limit, type):
    lim = limit or np.inf
    g, eg = product(x, wg, type)
    u, eu = product(x, wu, type)
    gc, uc = np.minimum(g, lim), np.clip(u, -lim, lim)
    h = R.act(a, gc) * uc
    tol = np.abs(uc) * (1.13 * eg + R._eval(gc)) + (np.abs(R.act(a, gc)) + 1.13 * eg) * eu
    return h, tol + HALF * np.abs(h) + 1e-38


def norm(s, gamma, eps):
    """(y before its rounding, the bound of y's error there, rstd)."""
    D = s.shape[1]
    rstd = 1 / np.sqrt((s * s).mean(1, keepdims=True) + eps)
    y = s * rstd * (1.0 if gamma is None else gamma)
    return y, ((D + 8) / 2 + 8) * U * np.abs(y) + 1e-38, rstd[:, 0]


def norm_backward(s, gamma, dy, ds, eps):
    """((dx, bound), (dgamma, bound)), both with their rounding to bf16."""
    M, D = s.shape
    r = 1 / np.sqrt((s * s).mean(1, keepdims=True) + eps)
    gd = dy * (1.0 if gamma is None else gamma)
    first, c = r * gd, (gd * s).sum(1, keepdims=True)
    dx = first - s * r ** 3 * c / D
    most = np.abs(s) * r ** 3 * np.abs(gd * s).sum(1, keepdims=True) / D
    tol = (D / 2 + 16) * U * np.abs(first) + (2.5 * D + 40) * U * most
    if ds is not None:
        dx = dx + ds
        tol = tol + 2 * U * (np.abs(ds) + np.abs(dx))
    dg, mag = (dy * s * r).sum(0), np.abs(dy * s * r).sum(0)
    return ((dx, tol + HALF * np.abs(dx) + 1e-38),
            (dg, (M + D / 2 + 32) * U * mag + HALF * np.abs(dg) + 1e-38))
