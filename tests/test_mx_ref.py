"""The 64-bit forms that the GPU tests of the norm and of microscaled values
compare with: known values, differences, and what the library refuses."""
import ctypes

import numpy as np
import pytest

import ffn_ref as R
import mx_ref as X


def test_the_types():
    assert X.E4M3[0x7E] == 448 and X.E4M3[1] == 2.0 ** -9 and X.E4M3[0x88] == -(2.0 ** -6) and np.isnan(X.E4M3[0xFF])
    assert list(X.E2M1[:8]) == [0, 0.5, 1, 1.5, 2, 3, 4, 6] and X.E2M1[15] == -6


@pytest.mark.parametrize("type", [X.MXFP8, X.MXFP4])
def test_quantize_known_values(type):
    v = np.zeros((1, 64))
    v[0, :8] = [6, 5, 2.5, 0.25, -0.75, 3.5, -1.25, 0.2500001]
    codes, scales = X.quantize(type, v)
    back = X.values(type, codes, scales)[0]
    if type == X.MXFP4:
        assert list(back[:8]) == [6, 4, 2, 0, -1, 4, -1, 0.5] and scales[0, 0] == 127
        assert codes[0, 0] == 7 | 6 << 4
    else:
        assert list(back[:7]) == list(v[0, :7]) and scales[0, 0] == 127 - 6     # 6 * 64 = 384 <= 448 < 768
    assert scales[0, 1] == 0 and not back[32:].any() and list(scales[0, 2:]) == [0, 0]


@pytest.mark.parametrize("type", [X.MXFP8, X.MXFP4])
def test_quantize_takes_the_least_scale(type):
    rng = np.random.default_rng(1)
    v = rng.standard_normal((50, 96)) * np.exp2(rng.integers(-40, 40, (50, 1)))
    codes, scales = X.quantize(type, v)
    top = np.abs(v).reshape(50, 3, 32).max(2)
    f = np.exp2(scales[:, :3] - 127.0)
    assert np.all(top <= X.MOST[type] * f) and np.all(top > X.MOST[type] * f / 2)
    d = np.abs(X.values(type, codes, scales) - v).reshape(50, 3, 32)
    step = 2.0 ** -4 * np.abs(v).reshape(50, 3, 32) + 2.0 ** -10 * f[..., None] if type == X.MXFP8 else f[..., None]
    assert np.all(d <= step)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_quantize_not_finite(bad):
    v = np.ones((1, 64))
    v[0, 40] = bad
    for type in (X.MXFP8, X.MXFP4):
        codes, scales = X.quantize(type, v)
        back = X.values(type, codes, scales)[0]
        assert np.all(back[:32] == 1) and np.all(np.isnan(back[32:])) and scales[0, 1] == 255
        assert not X.numbers(type, codes)[0, 32:].any()


@pytest.mark.parametrize("ds", [False, True])
@pytest.mark.parametrize("gain", [False, True])
def test_norm_gradient_by_differences(ds, gain):
    rng = np.random.default_rng(2)
    M, D, eps, h = 3, 17, 1e-3, 1e-6
    s, dy, add = rng.standard_normal((3, M, D))
    g = rng.standard_normal(D) if gain else None
    one = np.ones(D) if g is None else g

    def loss(s, g):
        return (X.norm(s, g, eps)[0] * dy).sum() + ((s * add).sum() if ds else 0.0)

    (dx, _), (dg, _) = X.norm_backward(s, g, dy, add if ds else None, eps)
    for m in range(M):
        for k in range(D):
            e = np.zeros((M, D))
            e[m, k] = h
            assert abs((loss(s + e, g) - loss(s - e, g)) / (2 * h) - dx[m, k]) < 1e-7
    for k in range(D):
        e = np.zeros(D)
        e[k] = h
        assert abs((loss(s, one + e) - loss(s, one - e)) / (2 * h) - dg[k]) < 1e-7


# ---- refusals: nothing here reaches a device --------------------------------

P = 1 << 20                                         # an aligned address that no call gets to read


def refused(lib, rc, *words):
    assert rc == 1
    said = lib.apus_ghip_last_error().decode()
    assert all(w in said for w in words), said


@pytest.fixture(scope="module")
def lib(pkg):
    return pkg.load()


def test_scale_rows(lib):
    assert [lib.apus_ghip_mx_scale_ld(k) for k in (32, 128, 160, 4096, 0)] == [4, 4, 8, 128, 0]


QUANT = dict(type=1, x=P, codes=P, scales=P, R=4, K=64, ldx=0)


@pytest.mark.parametrize("change,words", [
    (dict(type=0), ["type 0"]), (dict(type=3), ["type 3"]), (dict(x=None), ["x", "NULL"]), (dict(codes=None), ["codes", "NULL"]),
    (dict(scales=None), ["scales", "NULL"]), (dict(codes=P + 8), ["codes", "16-byte"]), (dict(scales=P + 2), ["scales", "4-byte"]),
    (dict(R=0), ["empty"]), (dict(K=0), ["empty"]), (dict(K=48), ["48", "32"]), (dict(ldx=63), ["ldx"]), (dict(R=1 << 31), ["large"])])
def test_quantize_refuses(lib, change, words):
    a = {**QUANT, **change}
    refused(lib, lib.apus_ghip_mx_quantize_dev(a["type"], a["x"], a["codes"], a["scales"], a["R"], a["K"], a["ldx"], None), *words)
    back = [w.replace("ldx", "ldo") for w in words if w != "x"]
    refused(lib, lib.apus_ghip_mx_dequant_dev(a["type"], a["codes"], a["scales"], a["x"], a["R"], a["K"], a["ldx"], None), *back)


NORM = dict(x=P, residual=P, gamma=P, sum=P, y=2 * P, codes=None, scales=None, rstd=None, M=4, D=64, ldx=0, ldr=0, lds=0, ldy=0, eps=1e-5)


@pytest.mark.parametrize("change,words", [
    (dict(x=None), ["x", "NULL"]), (dict(M=0), ["empty"]), (dict(D=0), ["empty"]), (dict(y=None), ["no output"]),
    (dict(residual=None), ["sum", "residual"]), (dict(y=P), ["same"]), (dict(eps=-1.0), ["eps"]), (dict(eps=float("nan")), ["eps"]),
    (dict(eps=float("inf")), ["eps"]), (dict(codes=P, scales=P, D=48), ["48", "32"]), (dict(codes=P), ["scales", "NULL"]),
    (dict(codes=P + 8, scales=P), ["codes", "16-byte"]), (dict(codes=P, scales=P + 1), ["scales", "4-byte"]),
    (dict(ldx=63), ["ldx"]), (dict(ldr=63), ["ldr"]), (dict(lds=63), ["lds"]), (dict(ldy=63), ["ldy"]), (dict(M=1 << 31), ["large"])])
def test_norm_refuses(lib, change, words):
    a = list({**NORM, **change}.values())
    refused(lib, lib.apus_ghip_rmsnorm_dev(*a, None), *words)


def grad_args(lib, **change):
    a = dict(s=P, gamma=P, rstd=P, dy=P, ds=None, dx=2 * P, dgamma=3 * P, M=4, D=64, lds=0, lddy=0, ldds=0, lddx=0, eps=1e-5, ws=4 * P,
             n=lib.apus_ghip_rmsnorm_backward_ws(4, 64))
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change,words", [
    (dict(s=None), ["s", "NULL"]), (dict(dy=None), ["dy", "NULL"]), (dict(dx=None, dgamma=None), ["no gradient"]), (dict(M=0), ["empty"]),
    (dict(eps=-0.5), ["eps"]), (dict(ws=None), ["workspace"]), (dict(ws=4 * P + 8), ["workspace"]), (dict(n=16), ["workspace"]),
    (dict(lds=1), ["lds"]), (dict(lddy=1), ["lddy"]), (dict(ldds=1), ["ldds"]), (dict(lddx=1), ["lddx"])])
def test_norm_backward_refuses(lib, change, words):
    refused(lib, lib.apus_ghip_rmsnorm_backward_dev(*grad_args(lib, **change), None), *words)


LIN = dict(w=P, ws=P, t=1, x=P, xs=P, bias=None, res=None, y=2 * P, M=4, O=24, K=64, ldx=0, ldr=0, ldy=0, act=0)


@pytest.mark.parametrize("change,words", [
    (dict(w=None), ["codes", "NULL"]), (dict(ws=None), ["scales", "NULL"]), (dict(x=None), ["x", "NULL"]), (dict(xs=None), ["scales", "NULL"]),
    (dict(y=None), ["output", "NULL"]), (dict(w=P + 4), ["codes", "16-byte"]), (dict(ws=P + 1), ["scales", "4-byte"]),
    (dict(x=P + 2), ["x", "16-byte"]), (dict(xs=P + 2), ["scales", "4-byte"]), (dict(t=3), ["type 3"]), (dict(t=-1), ["type -1"]),
    (dict(K=40), ["40", "32"]), (dict(M=0), ["empty"]), (dict(ldx=128), ["ldx 128", "dense"]), (dict(t=0, ldx=68), ["ldx 68", "8"]),
    (dict(t=0, ldx=32), ["ldx"]), (dict(ldr=8), ["ldr"]), (dict(ldy=8), ["ldy"]), (dict(act=5), ["activation"]),
    (dict(K=1 << 22), ["K 4194304", "long"]), (dict(t=0, K=1 << 22), ["long"]), (dict(t=0, ldx=1 << 22), ["ldx 4194304", "long"])])
def test_linear_refuses(lib, change, words):
    refused(lib, lib.apus_ghip_mxfp4_linear_dev(*{**LIN, **change}.values(), None), *words)


GATED = dict(wg=P, gs=P, wu=P, us=P, t=2, x=P, xs=P, h=2 * P, M=4, I=24, K=64, ldx=0, ldh=0, act=2, limit=0.0)


@pytest.mark.parametrize("change,words", [
    (dict(wg=None), ["codes", "NULL"]), (dict(wu=None), ["up codes", "NULL"]), (dict(us=None), ["up scales", "NULL"]),
    (dict(wu=P + 8), ["up codes", "16-byte"]), (dict(us=P + 2), ["up scales", "4-byte"]), (dict(limit=-1.0), ["limit"]),
    (dict(limit=float("nan")), ["limit"]), (dict(ldh=8), ["ldh"]), (dict(t=0, K=32800, ldx=1 << 22), ["ldx 4194304", "long"]), (dict(K=31), ["31", "32"])])
def test_gated_refuses(lib, change, words):
    refused(lib, lib.apus_ghip_mxfp4_gated_dev(*{**GATED, **change}.values(), None), *words)


def test_workspaces(lib):
    for M, O, K in [(1, 8, 32), (500, 2048, 4096), (33, 77, 96)]:
        assert lib.apus_ghip_mxfp4_linear_backward_ws(M, O, K) >= 2 * O * K + lib.apus_ghip_linear_ep_backward_ws(M, O, K)
        assert lib.apus_ghip_mxfp4_gated_backward_ws(M, O, K) >= 4 * O * K + lib.apus_ghip_gated_backward_ws(M, O, K)
    assert lib.apus_ghip_mxfp4_linear_backward_ws(4, 8, 40) == lib.apus_ghip_mxfp4_gated_backward_ws(0, 8, 32) == 0
    for M, D in [(1, 1), (300, 1536), (100000, 4096), (5, 70000)]:
        assert 4 * min(M, D) <= lib.apus_ghip_rmsnorm_backward_ws(M, D) <= 1 << 26
    assert lib.apus_ghip_rmsnorm_backward_ws(0, 8) == 0


@pytest.mark.parametrize("change,words", [
    (dict(w=None), ["codes", "NULL"]), (dict(dy=None), ["dy", "NULL"]), (dict(x=None, act=2), ["x", "NULL"]), (dict(dx=None), ["no gradient"]),
    (dict(ws=None), ["workspace"]), (dict(n=256), ["workspace"]), (dict(lddy=8), ["lddy"]), (dict(lddx=8), ["lddx"]), (dict(ldx=8), ["ldx"]),
    (dict(act=9), ["activation"]), (dict(K=33), ["33"])])
def test_linear_backward_refuses(lib, change, words):
    a = dict(w=P, s=P, x=P, bias=None, dy=P, dx=P, db=None, M=4, O=24, K=64, ldx=0, lddy=0, lddx=0, act=0, ws=P,
             n=lib.apus_ghip_mxfp4_linear_backward_ws(4, 24, 64))
    a.update(change)
    refused(lib, lib.apus_ghip_mxfp4_linear_backward_dev(*a.values(), None), *words)


@pytest.mark.parametrize("change,words", [
    (dict(wu=None), ["codes", "NULL"]), (dict(dh=None), ["dh", "NULL"]), (dict(x=None), ["x", "NULL"]), (dict(dx=None), ["dx", "NULL"]),
    (dict(ws=None), ["workspace"]), (dict(n=256), ["workspace"]), (dict(lddh=8), ["lddh"]), (dict(limit=-2.0), ["limit"])])
def test_gated_backward_refuses(lib, change, words):
    a = dict(wg=P, gs=P, wu=P, us=P, x=P, dh=P, dx=P, M=4, I=24, K=64, ldx=0, lddh=0, lddx=0, act=2, limit=0.0, ws=P,
             n=lib.apus_ghip_mxfp4_gated_backward_ws(4, 24, 64))
    a.update(change)
    refused(lib, lib.apus_ghip_mxfp4_gated_backward_dev(*a.values(), None), *words)
