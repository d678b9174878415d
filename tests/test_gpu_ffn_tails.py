"""The smooth activations and their slopes where they are small: relative to
their own value, from every kernel that computes them.

The bound, counted from what the kernels do:
  rounding   half a step of bf16, 2^-8 of the value.
  argument   exp's argument v is |z|, z^2 / 2 or 2 sqrt(2/pi) (|z| + 0.044715
             |z|^3), made of at most 8 roundings (the last, with the factor
             log2(e) of exp2): off by 8 * 2^-24 |v| relative, twice that for Phi
             (its other factors have arguments too). Times 4 where a slope adds
             terms of opposite sign (their sum is over 1/4 of the larger one for
             z <= -2).
  functions  Phi's polynomial, exp2, the reciprocal and the products around
             them: 2^-19 in all, times 4 as above.
  underflow  exp's and the reciprocal's results are 0 below 2^-126, and with
             them what multiplies them: 1 + |z| in the activation, 1 + |z| 2
             sqrt(2/pi) (1 + 3 * 0.044715 z^2) at most in a slope.
"""
import ctypes
import math

import numpy as np
import pytest

import ffn_forms as F
import ffn_ref as R
import gpu_util as G
from test_gpu_ffn import Mat, bf, ok, wide

pytestmark = pytest.mark.gpu

SMOOTH = [R.SILU, R.GELU, R.GELU_TANH]
K = 64
C, A = math.sqrt(2 / math.pi), 0.044715
_erfc = np.vectorize(math.erfc, otypes=[np.float64])


def points():
    """Every bf16 value of -32..-2, and fewer down to -100."""
    codes = np.arange(0xC000, 0xC200, dtype=np.uint16)
    return np.concatenate([wide(codes), wide(bf(-np.linspace(32.0, 100.0, 137)))])


def parts(a, z):
    """(sigmoid or Phi of z, the exponent behind it)."""
    if a == R.GELU:
        return 0.5 * _erfc(-z / math.sqrt(2)), z * z / 2
    v = np.abs(z) if a == R.SILU else 2 * C * (np.abs(z) + A * np.abs(z) ** 3)
    return np.exp(-v) / (1 + np.exp(-v)), v


def act(a, z):
    return z * parts(a, z)[0]


def slope(a, z):
    s, _ = parts(a, z)
    if a == R.GELU:
        return s + z * np.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if a == R.SILU:
        return s * (1 + z * (1 - s))
    return s * (1 + z * (1 - s) * 2 * C * (1 + 3 * A * z * z))


def bound(a, z, want, of):
    v = parts(a, z)[1] * (2 if a == R.GELU else 1)
    rel = 2.0 ** -8 + of * (2.0 ** -19 + v * 8 * 2.0 ** -24)
    return rel * np.abs(want) + 2.0 ** -126 * (1 + np.abs(z) * (1 if of == 1 else 2 * C * (1 + 3 * A * z * z)))


def near(got, a, z, of):
    """of: 1 the activation, 4 its slope."""
    want = (act if of == 1 else slope)(a, z)
    tol = bound(a, z, want, of)
    bad = np.flatnonzero(~(np.abs(got - want) <= tol))
    assert bad.size == 0, "act %d, %d of %d: z = %g gives %g, %g wanted" % (a, bad.size, z.size, z[bad[0]], got[bad[0]], want[bad[0]])


def column(M, N, at, values):
    m = np.zeros((M, N), np.float32)
    m[:, at] = values
    return G.dev(bf(m))


FORWARD = {"linear": F.LINEAR, "gated": F.GATED, "dlinear": F.DLINEAR, "dgated": F.DGATED}


@pytest.mark.parametrize("a", SMOOTH)
@pytest.mark.parametrize("route", ["tile", "rows", "any"])
@pytest.mark.parametrize("family", FORWARD)
def test_far_left(ghip, family, route, a):
    """x's column 0 holds z and column 1 holds 1; the (gate) weights pass the
    first on and the up projection's the second, exactly; the incoming gradient
    is 1."""
    mode, z = FORWARD[family], points()
    M, N = len(z), 16
    x = np.zeros((M, K), np.float32)
    x[:, 0], x[:, 1] = z, 1
    xd, w, u = G.dev(bf(x)), column(N, K, 0, 1.0), column(N, K, 1, 1.0)
    one, out, out2 = G.dev(bf(np.ones((M, N)))), Mat.out(M, N), Mat.out(M, N)
    at = lambda b: G.vp(b).value                                    # noqa: E731
    p = F.prod(family, M, N, K, a=at(xd), b=at(w), b2=at(u) if mode in (F.GATED, F.DGATED) else None)
    e = F.Ep(in_=at(one) if mode in (F.DLINEAR, F.DGATED) else None, out=out.p.value, out2=out2.p.value, ldin=N, ldout=N, act=a,
             limit=np.inf)
    if route == "tile":
        rc = ghip.ghip_launch_ffn_gemm(mode, 0, ctypes.c_uint32(1), ctypes.byref(p), ctypes.byref(e), None)
    elif route == "rows":
        rc = ghip.ghip_launch_ffn_rows(mode, 0, ctypes.byref(p), ctypes.byref(e), None)
    else:
        rc = ghip.ghip_launch_ffn_any(mode, ctypes.byref(p), ctypes.byref(e), None)
    assert rc == 0
    got = wide(out.get())
    assert np.all(got == got[:, :1])
    near(got[:, 0], a, z, 4 if mode in (F.DLINEAR, F.DGATED) else 1)
    if mode == F.DGATED:
        near(wide(out2.get())[:, 0], a, z, 1)


@pytest.mark.parametrize("a", SMOOTH)
def test_far_left_of_the_entries(ghip, a):
    """One row of x, z in the weights: y, dw and dbias of linear_ep."""
    z = points()
    N = len(z)
    x, w, y = Mat(bf(np.eye(1, K))), column(N, K, 0, z), Mat.out(1, N)
    ok(ghip, ghip.apus_ghip_bf16_linear_ep_dev(G.vp(w), x.p, None, None, y.p, 1, N, K, 0, 0, 0, a, None))
    near(wide(y.get())[0], a, z, 1)
    dy, dw, db = Mat(bf(np.ones((1, N)))), Mat.out(N, K), Mat.out(1, N)
    need = ghip.apus_ghip_linear_ep_backward_ws(1, N, K)
    ws = G.empty(need)
    ok(ghip, ghip.apus_ghip_bf16_linear_ep_backward_dev(G.vp(w), x.p, None, dy.p, None, dw.p, db.p, 1, N, K, 0, 0, 0, a, G.vp(ws),
                                                         need, None))
    near(wide(db.get())[0], a, z, 4)
    near(wide(dw.get())[:, 0], a, z, 4)
