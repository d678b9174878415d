"""ReLU's gradients where something is not finite: none passes where z <= 0,
whatever comes in, and a NaN z stays one, as in the forward."""
import ctypes

import numpy as np
import pytest

import ffn_forms as F
import ffn_ref as R
import gpu_util as G
from test_gpu_ffn import Mat, bf, ok, wide

pytestmark = pytest.mark.gpu

K, N = 64, 16
Z = [-3.0, -0.0, 0.0, 2.0, -np.inf, np.inf, np.nan]
IN = [1.5, np.inf, -np.inf, np.nan, 0.0]


def wanted(z, d):
    """dz of z and the incoming gradient d."""
    return np.where(np.isnan(z), np.nan, np.where(z > 0, d, 0.0))


def grid(copies):
    z, d = (np.tile(v.ravel(), copies) for v in np.meshgrid(Z, IN))
    return z, d


def launch(lib, route, mode, p, e):
    if route == "tile":
        return lib.ghip_launch_ffn_gemm(mode, 0, ctypes.c_uint32(1), ctypes.byref(p), ctypes.byref(e), None)
    if route == "rows":
        return lib.ghip_launch_ffn_rows(mode, 0, ctypes.byref(p), ctypes.byref(e), None)
    return lib.ghip_launch_ffn_any(mode, ctypes.byref(p), ctypes.byref(e), None)


def at(b):
    return G.vp(b).value


def same(got, want):
    """-0 is 0"""
    assert np.array_equal(got, np.broadcast_to(want[:, None], got.shape), equal_nan=True), (got[:, 0], want)


@pytest.mark.parametrize("route", ["tile", "rows", "any"])
def test_dz(ghip, route):
    """z comes from the bias: a sum of 0 plus it."""
    z, d = grid(1)
    M, n = 9, len(z)
    w, x, bias = G.dev(np.zeros((n, K), np.uint16)), G.dev(np.zeros((M, K), np.uint16)), G.dev(bf(z))
    dy, out = G.dev(bf(np.tile(d, (M, 1)))), Mat.out(M, n)
    p = F.prod("dlinear", M, n, K, a=at(x), b=at(w))
    e = F.Ep(bias=at(bias), in_=at(dy), out=out.p.value, ldin=n, ldout=n, act=R.RELU, limit=np.inf)
    assert launch(ghip, route, F.DLINEAR, p, e) == 0
    same(wide(out.get()).T, wanted(wide(bf(z)), d))


@pytest.mark.parametrize("route", ["tile", "rows", "any"])
def test_dg(ghip, route):
    """g of x's column 0 (not the infinite ones: 0 * inf in the other products),
    u = 1."""
    z, d = grid(1)
    z, d = z[np.isfinite(z)], d[np.isfinite(z)]
    M = len(z)
    x = np.zeros((M, K), np.float32)
    x[:, 0], x[:, 1] = z, 1
    wg, wu = np.zeros((N, K), np.float32), np.zeros((N, K), np.float32)
    wg[:, 0] = wu[:, 1] = 1
    xd, g, u, dh = G.dev(bf(x)), G.dev(bf(wg)), G.dev(bf(wu)), G.dev(bf(np.tile(d[:, None], (1, N))))
    out, out2 = Mat.out(M, N), Mat.out(M, N)
    p = F.prod("dgated", M, N, K, a=at(xd), b=at(g), b2=at(u))
    e = F.Ep(in_=at(dh), out=out.p.value, out2=out2.p.value, ldin=N, ldout=N, act=R.RELU, limit=np.inf)
    assert launch(ghip, route, F.DGATED, p, e) == 0
    same(wide(out.get()), wanted(z, d))


def test_through_the_entry(ghip):
    """An infinite dy at closed units only: dw is that of the open ones, dbias 0
    there."""
    rng = np.random.default_rng(5)
    M, n = 40, 24
    x = rng.uniform(0.5, 1.5, (M, K))
    w = rng.uniform(0.5, 1.0, (n, K)) * np.where(np.arange(n) % 3 == 0, -1, 1)[:, None]
    dy = rng.standard_normal((M, n))
    dy[:, ::3] = np.inf
    xb, wb, db_ = bf(x), bf(w), bf(dy)
    xd, wd, dd = Mat(xb), G.dev(wb), Mat(db_)
    dx, dw, db = Mat.out(M, K), Mat.out(n, K), Mat.out(1, n)
    need = ghip.apus_ghip_linear_ep_backward_ws(M, n, K)
    ws = G.empty(need)
    ok(ghip, ghip.apus_ghip_bf16_linear_ep_backward_dev(G.vp(wd), xd.p, None, dd.p, dx.p, dw.p, db.p, M, n, K, 0, 0, 0, R.RELU, G.vp(ws),
                                                         need, None))
    finite = np.where(np.isfinite(wide(db_)), wide(db_), 0.0)
    want = R.linear_backward(wide(xb), wide(wb), None, finite, R.RELU)
    R.check(wide(dx.get()), *want["dx"], "dx")
    R.check(wide(dw.get()), *want["dw0"], "dw")
    R.check(wide(db.get())[0], *want["db"], "db")
