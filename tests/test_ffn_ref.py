"""The 64-bit forms of tests/ffn_ref.py against differences, and the refusals
of the dense feed-forward entries (arguments are checked before any device)."""
import ctypes

import numpy as np
import pytest

import ffn_ref as R

P = ctypes.c_void_p(1 << 20)


@pytest.mark.parametrize("a", R.ACTS)
def test_slopes_are_the_activations_differences(a):
    z = np.linspace(-9, 9, 2000)                                    # no point at relu's corner
    e = 1e-5
    assert np.max(np.abs((R.act(a, z + e) - R.act(a, z - e)) / (2 * e) - R.slope(a, z))) < 1e-8


@pytest.mark.parametrize("a", [R.SILU, R.GELU, R.GELU_TANH])
def test_slopes_and_curvatures_stay_under_the_bounds(a):
    z = np.linspace(-30, 30, 60001)
    s = R.slope(a, z)
    assert np.max(np.abs(s)) <= 1.13 and np.max(np.abs(np.diff(s) / np.diff(z))) <= 1.1


@pytest.mark.parametrize("a", R.ACTS)
@pytest.mark.parametrize("limit", [0.0, 0.8])
def test_gated_gradients_are_differences(a, limit):
    rng = np.random.default_rng(3)
    x, wg, wu, dh = (rng.standard_normal(s) * 0.7 for s in ((5, 6), (4, 6), (4, 6), (5, 4)))
    got = R.gated_backward(x, wg, wu, dh, a, limit)
    loss = lambda: float(np.sum(dh * R.gated(x, wg, wu, a, limit)[0]))  # noqa: E731
    for t, key in ((x, "dx"), (wg, "dw0"), (wu, "dw1")):
        for i in np.ndindex(*t.shape):
            v = t[i]
            t[i] = v + 1e-6
            hi = loss()
            t[i] = v - 1e-6
            lo = loss()
            t[i] = v
            assert abs((hi - lo) / 2e-6 - got[key][0][i]) < 1e-6


@pytest.mark.parametrize("a", R.ACTS)
def test_linear_gradients_are_differences(a):
    rng = np.random.default_rng(4)
    x, w, b, dy = (rng.standard_normal(s) * 0.7 for s in ((5, 6), (4, 6), (4,), (5, 4)))
    got = R.linear_backward(x, w, b, dy, a)
    loss = lambda: float(np.sum(dy * R.linear(x, w, b, None, a)[0]))  # noqa: E731
    for t, key in ((x, "dx"), (w, "dw0"), (b, "db")):
        for i in np.ndindex(*t.shape):
            v = t[i]
            t[i] = v + 1e-6
            hi = loss()
            t[i] = v - 1e-6
            lo = loss()
            t[i] = v
            assert abs((hi - lo) / 2e-6 - got[key][0][i]) < 1e-6


BIG = 1 << 31
NAN = float("nan")


def linear(lib, w=P, x=P, b=P, r=P, y=P, M=4, O=16, K=32, ldx=0, ldr=0, ldy=0, act=0):
    return lib.apus_ghip_bf16_linear_ep_dev(w, x, b, r, y, M, O, K, ldx, ldr, ldy, act, None)


def linear8(lib, c=P, s=P, x=P, b=P, r=P, y=P, M=4, O=16, K=32, ldx=0, ldr=0, ldy=0, act=0, exact=0):
    return lib.apus_ghip_fp8blk_linear_ep_dev(c, s, x, b, r, y, M, O, K, ldx, ldr, ldy, act, exact, None)


def gated(lib, wg=P, wu=P, x=P, h=P, M=4, I=16, K=32, ldx=0, ldh=0, act=2, limit=0.0):
    return lib.apus_ghip_bf16_gated_dev(wg, wu, x, h, M, I, K, ldx, ldh, act, limit, None)


def gated8(lib, cg=P, sg=P, cu=P, su=P, x=P, h=P, M=4, I=16, K=32, ldx=0, ldh=0, act=2, limit=0.0, exact=0):
    return lib.apus_ghip_fp8blk_gated_dev(cg, sg, cu, su, x, h, M, I, K, ldx, ldh, act, limit, exact, None)


def linear_bwd(lib, w=P, x=P, b=P, dy=P, dx=P, dw=P, db=P, M=4, O=16, K=32, ldx=0, lddy=0, lddx=0, act=2, ws=P, n=1 << 20):
    return lib.apus_ghip_bf16_linear_ep_backward_dev(w, x, b, dy, dx, dw, db, M, O, K, ldx, lddy, lddx, act, ws, n, None)


def gated_bwd(lib, wg=P, wu=P, x=P, dh=P, dx=P, dwg=P, dwu=P, M=4, I=16, K=32, ldx=0, lddh=0, lddx=0, act=2, limit=0.0,
              ws=P, n=1 << 20):
    return lib.apus_ghip_bf16_gated_backward_dev(wg, wu, x, dh, dx, dwg, dwu, M, I, K, ldx, lddh, lddx, act, limit, ws, n, None)


REFUSED = [
    (linear, [dict(w=None), dict(x=None), dict(y=None), dict(M=0), dict(O=0), dict(K=0), dict(M=BIG), dict(O=BIG), dict(K=BIG),
              dict(ldx=31), dict(ldr=15), dict(ldy=15), dict(ldx=BIG), dict(act=-1), dict(act=5)]),
    (linear8, [dict(c=None), dict(s=None), dict(x=None), dict(y=None), dict(M=0), dict(ldx=31), dict(ldy=15), dict(act=9)]),
    (gated, [dict(wg=None), dict(wu=None), dict(x=None), dict(h=None), dict(M=0), dict(I=0), dict(K=0), dict(ldx=31), dict(ldh=15),
             dict(act=5), dict(limit=-1.0), dict(limit=NAN)]),
    (gated8, [dict(cg=None), dict(sg=None), dict(cu=None), dict(su=None), dict(x=None), dict(h=None), dict(I=0), dict(limit=NAN)]),
    (linear_bwd, [dict(w=None), dict(x=None), dict(dy=None), dict(dx=None, dw=None, db=None), dict(M=0), dict(ldx=31), dict(lddy=15),
                  dict(lddx=31), dict(act=5), dict(ws=None), dict(ws=ctypes.c_void_p((1 << 20) + 8)), dict(n=4 * 16 * 2 - 1),
                  dict(act=0, w=None), dict(act=0, x=None)]),
    (gated_bwd, [dict(wg=None), dict(wu=None), dict(x=None), dict(dh=None), dict(dx=None, dwg=None, dwu=None), dict(K=0), dict(ldx=31),
                 dict(lddh=15), dict(lddx=31), dict(act=-2), dict(limit=-0.5), dict(ws=None), dict(n=2 * 256 - 1)]),
]


@pytest.mark.parametrize("call,args", [(c, a) for c, many in REFUSED for a in many],
                         ids=lambda v: v.__name__ if callable(v) else "-".join(v))
def test_refusals_come_before_the_device(pkg, call, args):
    lib = pkg.load()
    assert call(lib, **args) == 1
    said = lib.apus_ghip_last_error().decode()
    assert said and "device" not in said and "hip" not in said.lower(), said


def test_workspace_sizes(pkg):
    """dz's matrix (two of them), in whole 256 bytes, and the partial sums of the
    products that may be split: at most 16 times the outputs and 32 MiB."""
    lib = pkg.load()
    one, two = lib.apus_ghip_linear_ep_backward_ws, lib.apus_ghip_gated_backward_ws
    assert one(4, 16, 32) == 256 and two(4, 16, 32) == 512          # 4 rows of 32 bytes
    assert one(3, 9, 5) == 256 and one(100, 9, 5) == 3328            # rows of 9 take 16 elements
    # outputs of 2^20 x 8 (dx) over 2^14, of 2^14 x 8 (dW) over 2^20
    assert one(1 << 20, 1 << 14, 8) == (1 << 35) + 16 * (1 << 17) * 4
    # dx: 16 x 64 outputs over 8192 split 16 times; over 2 x 8192 the same
    assert one(16, 8192, 64) == 16 * 8192 * 2 + 16 * 16 * 64 * 4
    assert two(16, 8192, 64) == 2 * 16 * 8192 * 2 + 16 * 16 * 64 * 4
    assert [f(*s) for f in (one, two) for s in ((0, 1, 1), (1, 0, 1), (1, 1, 0), (BIG, 1, 1), (1, 1, BIG))] == [0] * 10
