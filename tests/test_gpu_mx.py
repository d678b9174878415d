"""Microscaled values and the products with MXFP4 weights on the device against
tests/mx_ref.py's 64-bit forms: every code and scale, shapes of every route,
strides, values that are not finite, streams, graphs, and a block of norm,
products and quantization as it is used."""
import numpy as np
import pytest

import ffn_ref as R
import gpu_util as G
import mx_ref as X
import oracle as O
from test_gpu_ffn import Mat, bf, ok, seed, wide
from test_gpu_norm import Bytes

pytestmark = pytest.mark.gpu

TYPES = [X.MXFP8, X.MXFP4]
XTYPES = [X.BF16, X.MXFP8, X.MXFP4]


class Mx:
    """Microscaled rows on the device, from codes and scales as stored."""

    def __init__(self, type, codes, scales):
        self.type, self.codes, self.scales = type, G.dev(codes), G.dev(scales)
        self.values = X.values(type, codes, scales)

    @classmethod
    def of(cls, type, v):
        return cls(type, *X.quantize(type, v))


def quantize(lib, type, x, st=None):
    c, s = Bytes(x.rows, x.cols // (1 if type == X.MXFP8 else 2)), Bytes(x.rows, X.scale_ld(x.cols))
    ok(lib, lib.apus_ghip_mx_quantize_dev(type, x.p, c.p, s.p, x.rows, x.cols, x.ld, st))
    return c.get(), s.get()


MX_SHAPES = [(1, 32), (1, 4096), (3, 64), (2, 96), (5, 160), (33, 2048), (257, 1120), (1111, 2048), (1, 65536), (4100, 32)]


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("Rr,K", MX_SHAPES)
def test_quantize_and_back(ghip, Rr, K, type):
    """Bitwise, both ways; blocks of zeros, of one value, of values of all magnitudes; -0 keeps its sign."""
    rng = seed(41, Rr, K, type)
    v = rng.standard_normal((Rr, K)) * np.exp2(rng.integers(-30, 30, (Rr, 1)))
    v[:, :32] *= np.exp2(rng.integers(-12, 3, (Rr, 32)))
    if K > 32:
        v[0, 32:64] = 0
        v[Rr - 1, 40] = -0.0
    x = bf(v)
    for pad, off in ((0, 0), (8, 8), (3, 1)):
        codes, scales = quantize(ghip, type, Mat(x, pad, off, 0x7FC0))
        want, wscales = X.quantize(type, wide(x))
        assert np.array_equal(scales, wscales) and np.array_equal(codes, want)
        out = Mat.out(Rr, K, pad, off)
        q = Mx(type, codes, scales)
        ok(ghip, ghip.apus_ghip_mx_dequant_dev(type, G.vp(q.codes), G.vp(q.scales), out.p, Rr, K, out.ld, None))
        assert np.array_equal(wide(out.get()), q.values)


@pytest.mark.parametrize("type", TYPES)
def test_every_code_and_scale_read_back(ghip, type):
    n = 256 if type == X.MXFP8 else 32
    c = np.tile((np.arange(n) % (256 if n == 256 else 16)).astype(np.uint8), (256, 1))
    codes, scales = X.stored(type, c), np.zeros((256, X.scale_ld(n)), np.uint8)
    scales[:, :n // 32] = np.arange(256)[:, None]
    out = Mat.out(256, n)
    q = Mx(type, codes, scales)
    ok(ghip, ghip.apus_ghip_mx_dequant_dev(type, G.vp(q.codes), G.vp(q.scales), out.p, 256, n, 0, None))
    with np.errstate(over="ignore"):
        want = O.bf16_to_f32(bf(q.values.astype(np.float32)))
    got = O.bf16_to_f32(out.get())
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(got[~np.isnan(want)], want[~np.isnan(want)])


@pytest.mark.parametrize("type", TYPES)
def test_quantize_at_the_borders(ghip, type):
    """Blocks whose largest value is at, below and above the type's largest; every tie between two numbers; the largest and
    least bf16 values; blocks with a NaN or an infinity."""
    rows = []
    grid = X.E4M3[:127] if type == X.MXFP8 else X.E2M1[:8]
    most = X.MOST[type]
    for top in (most, most * (1 + 2.0 ** -7), most * (1 - 2.0 ** -8), most / 2):
        for e in (-120, -3, 0, 50):
            rows.append([top * 2.0 ** e] + [0.1 * 2.0 ** e * k for k in range(31)])
    mid = (grid[1:] + grid[:-1]) / 2
    for k in range(0, len(mid), 15):
        part = np.concatenate([mid[k:k + 15], -mid[k:k + 15]])
        rows.append([most] + list(part) + [0] * (31 - len(part)))
    rows += [[3.3e38] * 32, [2.0 ** -133] + [0] * 31, [-(2.0 ** -126)] * 32]
    x = bf(np.array(rows, np.float64))
    for bad in (0x7FC0, 0x7F80, 0xFF80):
        r = bf(np.ones((1, 32)))
        r[0, 9] = bad
        x = np.concatenate([x, r])
    codes, scales = quantize(ghip, type, Mat(x))
    with np.errstate(invalid="ignore"):
        want, wscales = X.quantize(type, wide(x))
    assert np.array_equal(scales, wscales) and np.array_equal(codes, want)
    assert np.all(scales[-3:, 0] == 255) and not codes[-3:].any()


def test_more_pieces_than_32_bits_of_one_launch_take(ghip):
    """2^33 values: rows past the first launch's are quantized and read back."""
    Rr, K = (1 << 21) + 5, 4096
    x, c, s = G.empty(2 * Rr * K), G.empty(Rr * K // 2), G.empty(Rr * X.scale_ld(K))
    ok(ghip, ghip.apus_synth_bf16_normal_dev(G.vp(x), Rr * K, 5, 6, 0, None))
    ok(ghip, ghip.apus_ghip_mx_quantize_dev(X.MXFP4, G.vp(x), G.vp(c), G.vp(s), Rr, K, 0, None))
    rows = (0, (1 << 21) - 2, 1 << 21, Rr - 1)
    want = []
    for r in rows:
        q = X.quantize(X.MXFP4, wide(G.download_ptr(x.ptr + 2 * r * K, np.uint16, (1, K))))
        assert np.array_equal(G.download_ptr(c.ptr + r * K // 2, np.uint8, (1, K // 2)), q[0])
        assert np.array_equal(G.download_ptr(s.ptr + r * X.scale_ld(K), np.uint8, (1, X.scale_ld(K))), q[1])
        want.append(X.values(X.MXFP4, *q))
    ok(ghip, ghip.apus_ghip_mx_dequant_dev(X.MXFP4, G.vp(c), G.vp(s), G.vp(x), Rr, K, 0, None))
    for r, w in zip(rows, want):
        assert np.array_equal(wide(G.download_ptr(x.ptr + 2 * r * K, np.uint16, (1, K))), w)


# ---- products -----------------------------------------------------------------

SHAPES = [(1, 1, 32), (1, 5, 64), (1, 300, 2048), (1, 4096, 4096), (2, 4096, 128), (3, 257, 96), (4, 1000, 4096), (5, 96, 160), (9, 77, 224),
          (7, 2050, 640), (8, 129, 1536), (13, 64, 64), (16, 768, 192), (17, 33, 32), (31, 520, 992), (33, 1025, 576), (64, 512, 1024),
          (65, 255, 96), (100, 2048, 512), (129, 130, 288), (200, 1537, 320), (255, 257, 256), (256, 256, 64), (300, 520, 1088),
          (513, 1032, 160), (700, 2049, 192), (1111, 640, 448), (2049, 1030, 256)]


class Act:
    """x of one of the three types."""

    def __init__(self, xt, x, pad=0, off=0):
        """x: bf16 codes; microscaled rows are dense."""
        self.type = xt
        if xt == X.BF16:
            self.mat = Mat(x, pad, off, 0x7FC0)
            self.args, self.ld, self.values = (xt, self.mat.p, None), self.mat.ld, wide(x)
        else:
            self.mx = Mx.of(xt, wide(x))
            self.args, self.ld, self.values = (xt, G.vp(self.mx.codes), G.vp(self.mx.scales)), 0, self.mx.values


def weights(rng, N, K, scale=1.0):
    return Mx.of(X.MXFP4, rng.standard_normal((N, K)) * scale / np.sqrt(K))


def acts(rng, M, K):
    return bf(rng.standard_normal((M, K)) * (1 + 9 * (rng.random(K) < 0.02)))


def linear(lib, w, x, bias, res, y, act, st=None):
    M, N, K = y.rows, y.cols, w.values.shape[1]
    return lib.apus_ghip_mxfp4_linear_dev(G.vp(w.codes), G.vp(w.scales), *x.args, None if bias is None else G.vp(bias),
                                          None if res is None else res.p, y.p, M, N, K, x.ld, 0 if res is None else res.ld, y.ld, act, st)


def gated(lib, wg, wu, x, h, act, limit, st=None):
    M, N, K = h.rows, h.cols, wg.values.shape[1]
    return lib.apus_ghip_mxfp4_gated_dev(G.vp(wg.codes), G.vp(wg.scales), G.vp(wu.codes), G.vp(wu.scales), *x.args, h.p, M, N, K, x.ld,
                                         h.ld, act, limit, st)


@pytest.mark.parametrize("xt", XTYPES)
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear(ghip, M, N, K, xt):
    i = SHAPES.index((M, N, K))
    rng, act = seed(42, M, N, K, xt), R.ACTS[(i + xt) % 5]
    w, x = weights(rng, N, K), Act(xt, acts(rng, M, K))
    bias = bf(rng.standard_normal(N)) if (i + xt) % 2 else None
    res = bf(rng.standard_normal((M, N))) if (i + xt) % 3 else None
    y = Mat.out(M, N, off=8)
    ok(ghip, linear(ghip, w, x, None if bias is None else G.dev(bias), None if res is None else Mat(res), y, act))
    R.check(wide(y.get()), *X.linear(x.values, w.values, None if bias is None else wide(bias), None if res is None else wide(res), act, xt),
            "linear")


@pytest.mark.parametrize("xt", XTYPES)
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_gated(ghip, M, N, K, xt):
    i = SHAPES.index((M, N, K))
    rng, act, limit = seed(43, M, N, K, xt), R.ACTS[(i + 2 + xt) % 5], (0.0, 1.5)[i % 2]
    wg, wu, x = weights(rng, N, K), weights(rng, N, K), Act(xt, acts(rng, M, K))
    h = Mat.out(M, N, off=8)
    ok(ghip, gated(ghip, wg, wu, x, h, act, limit))
    R.check(wide(h.get()), *X.gated(x.values, wg.values, wu.values, act, limit, xt), "gated")


@pytest.mark.parametrize("xt", XTYPES)
@pytest.mark.parametrize("M,N,K", [(1, 520, 512), (6, 264, 96), (40, 392, 384), (300, 520, 640), (300, 517, 1120)])
@pytest.mark.parametrize("pad,off", [(8, 8), (64, 0), (3, 1), (1, 3)])
def test_rows_in_wider_buffers(ghip, M, N, K, xt, pad, off):
    """Residual and outputs of any alignment, BF16 x of whole 16 bytes; the columns between hold NaN and stay."""
    rng = seed(44, M, N, K, xt)
    w, w2, x = weights(rng, N, K), weights(rng, N, K), Act(xt, acts(rng, M, K), (pad + 7) // 8 * 8, off // 8 * 8)
    res, bias = bf(rng.standard_normal((M, N))), bf(rng.standard_normal((1, N)))
    y, h = Mat.out(M, N, pad, off), Mat.out(M, N, pad, off)
    b, r = Mat(bias, 0, off), Mat(res, pad, off, 0x7FC0)
    ok(ghip, ghip.apus_ghip_mxfp4_linear_dev(G.vp(w.codes), G.vp(w.scales), *x.args, b.p, r.p, y.p, M, N, K, x.ld, r.ld, y.ld, R.NONE, None))
    R.check(wide(y.get()), *X.linear(x.values, w.values, wide(bias), wide(res), R.NONE, xt), "linear")
    ok(ghip, gated(ghip, w, w2, x, h, R.SILU, 2.0))
    R.check(wide(h.get()), *X.gated(x.values, w.values, w2.values, R.SILU, 2.0, xt), "gated")


@pytest.mark.parametrize("xt", XTYPES)
def test_long_k(ghip, xt):
    """A row of x longer than LDS: few rows go to tiles."""
    M, N, K = 3, 40, (1 << 17) + 96
    rng = seed(50, xt)
    w, x, y = weights(rng, N, K), Act(xt, acts(rng, M, K)), Mat.out(M, N)
    ok(ghip, linear(ghip, w, x, None, None, y, R.NONE))
    R.check(wide(y.get()), *X.linear(x.values, w.values, None, None, R.NONE, xt), "linear")


@pytest.mark.parametrize("xt", XTYPES)
@pytest.mark.parametrize("M,N,K", [(4, 512, 1024), (300, 520, 640), (1024, 1032, 256), (5000, 2056, 128)])
def test_called_again(ghip, M, N, K, xt):
    """The same bits from call to call, many workgroups a CU among them."""
    rng = seed(51, M, N, K, xt)
    w, x, res = weights(rng, N, K), Act(xt, acts(rng, M, K)), Mat(bf(rng.standard_normal((M, N))))
    first = None
    for _ in range(4):
        y = Mat.out(M, N)
        ok(ghip, linear(ghip, w, x, None, res, y, R.NONE))
        got = y.get()
        assert first is None or np.array_equal(first, got)
        first = got


@pytest.mark.parametrize("xt", XTYPES)
@pytest.mark.parametrize("M,N,K", [(1, 4096, 1024), (9, 1040, 512), (333, 777, 192)])
def test_residual_in_place(ghip, M, N, K, xt):
    rng = seed(45, M, N, K, xt)
    w, x, res = weights(rng, N, K), Act(xt, acts(rng, M, K)), bf(rng.standard_normal((M, N)))
    y, other = Mat(res, 8, 8), Mat.out(M, N)
    ok(ghip, linear(ghip, w, x, None, y, y, R.GELU))
    ok(ghip, linear(ghip, w, x, None, Mat(res), other, R.GELU))
    assert np.array_equal(y.get(), other.get())


@pytest.mark.parametrize("xt", XTYPES)
@pytest.mark.parametrize("M", [1, 3, 40, 300])
@pytest.mark.parametrize("K", [96, 128, 512])
def test_not_finite_values_stay_in_their_rows(ghip, M, K, xt):
    """A NaN in x's last row (a NaN block where it is microscaled), a NaN block in w's last row, an infinity in the residual
    reach exactly their own row, column and element."""
    N = 265
    rng = seed(46, M, K, xt)
    v = rng.uniform(1, 2, (N, K))
    v[N - 1, K - 1] = np.nan
    x, res = bf(rng.uniform(1, 2, (M, K))), bf(rng.standard_normal((M, N)))
    x[M - 1, K - 2], res[0, 2] = 0x7FC0, 0xFF80
    with np.errstate(invalid="ignore"):
        w, a = Mx.of(X.MXFP4, v), Act(xt, x)
    y = Mat.out(M, N)
    ok(ghip, linear(ghip, w, a, None, Mat(res), y, R.NONE))
    got = O.bf16_to_f32(y.get())
    assert np.all(np.isnan(got[:, N - 1])) and np.all(np.isnan(got[M - 1]))
    if M > 1:
        assert np.isneginf(got[0, 2])
        got[0, 2] = 0
        assert np.all(np.isfinite(got[:M - 1, :N - 1]))


@pytest.mark.parametrize("xt", TYPES)
@pytest.mark.parametrize("M,N", [(2, 40), (130, 300)])
def test_scales_of_every_size(ghip, M, N, xt):
    """Blocks of x from 2^-127 on and of w up to 2^120, whose products are ordinary numbers; one of each row alone counts."""
    K = 256
    rng = seed(47, M, N, xt)
    cx = rng.integers(0, 256 if xt == X.MXFP8 else 16, (M, K)).astype(np.uint8)
    if xt == X.MXFP8:
        cx[cx & 0x7F == 0x7F] = 0
    cw = rng.integers(0, 16, (N, K)).astype(np.uint8)
    e = np.array([0, 1, 7, 60, 127, 200, 246, 254])
    sx, sw = np.zeros((M, 8), np.uint8), np.zeros((N, 8), np.uint8)
    sx[:], sw[:] = e, np.minimum(254 - e, 246)
    w, x = Mx(X.MXFP4, X.stored(X.MXFP4, cw), sw), Act.__new__(Act)
    x.mx = Mx(xt, X.stored(xt, cx), sx)
    x.type, x.args, x.ld, x.values = xt, (xt, G.vp(x.mx.codes), G.vp(x.mx.scales)), 0, x.mx.values
    y = Mat.out(M, N)
    ok(ghip, linear(ghip, w, x, None, None, y, R.NONE))
    R.check(wide(y.get()), *X.linear(x.values, w.values, None, None, R.NONE, xt), "linear")


@pytest.mark.parametrize("M,N,K", [(3, 520, 96), (40, 200, 1056), (300, 777, 160), (300, 130, 32), (300, 130, 96)])
def test_bytes_behind_the_last_scale_are_not_read(ghip, M, N, K):
    """The scale rows' words behind K's last block hold NaN scales."""
    rng = seed(48, M, N, K)
    x = acts(rng, M, K)
    for xt in XTYPES:
        w, a = weights(rng, N, K), Act(xt, x)
        y = [Mat.out(M, N) for _ in range(2)]
        ok(ghip, linear(ghip, w, a, None, None, y[0], R.NONE))
        for m in (w, a.mx) if xt else (w,):
            s = m.scales.download(np.uint8, (m.values.shape[0], X.scale_ld(K)))
            s[:, K // 32:] = 255
            m.scales.upload(s)
        ok(ghip, linear(ghip, w, a, None, None, y[1], R.NONE))
        assert np.array_equal(y[0].get(), y[1].get())


BWD = [(1, 40, 32), (5, 264, 96), (40, 392, 384), (300, 520, 1088), (500, 1030, 256), (130, 77, 64)]


def run_linear_bwd(lib, w, x, bias, dy, act, want=("dx", "db"), st=None, pad=0):
    (M, N), K = (dy.rows, dy.cols), w.values.shape[1]
    out = {"dx": Mat.out(M, K, pad, 8), "db": Mat.out(1, N, 0, 8)}
    need = lib.apus_ghip_mxfp4_linear_backward_ws(M, N, K)
    ws = Mat.out(1, need // 2)
    p = lambda k: out[k].p if k in want else None  # noqa: E731
    ok(lib, lib.apus_ghip_mxfp4_linear_backward_dev(G.vp(w.codes), G.vp(w.scales), None if x is None else x.p,
                                                    None if bias is None else G.vp(bias), dy.p, p("dx"), p("db"), M, N, K,
                                                    0 if x is None else x.ld, dy.ld, out["dx"].ld, act, ws.p, need, st))
    got = {k: m.get() for k, m in out.items()}
    ws.get()
    return got


@pytest.mark.parametrize("M,N,K", BWD)
def test_linear_backward(ghip, M, N, K):
    for act in R.ACTS:
        rng = seed(49, M, N, K, act)
        w, x, dy = weights(rng, N, K), acts(rng, M, K), bf(rng.standard_normal((M, N)))
        bias = bf(rng.standard_normal(N)) if act % 2 else None
        got = run_linear_bwd(ghip, w, None if act == R.NONE else Mat(x, 8, 8), None if bias is None else G.dev(bias), Mat(dy, 3, 1), act, pad=5)
        want = R.linear_backward(wide(x), w.values, None if bias is None else wide(bias), wide(dy), act)
        R.check(wide(got["dx"]), *want["dx"], "dx")
        R.check(wide(got["db"])[0], *want["db"], "db")
        one = run_linear_bwd(ghip, w, None if act == R.NONE else Mat(x, 8, 8), None if bias is None else G.dev(bias), Mat(dy, 3, 1), act, ("db",))
        assert np.array_equal(one["db"], got["db"]) and np.all(one["dx"] == 0x7E57)


@pytest.mark.parametrize("M,N,K", BWD)
def test_gated_backward(ghip, M, N, K):
    for act, limit in ((R.SILU, 1.5), (R.GELU_TANH, 0.0)):
        rng = seed(50, M, N, K, act)
        wg, wu, x, dh = weights(rng, N, K), weights(rng, N, K), acts(rng, M, K), bf(rng.standard_normal((M, N)))
        dx, xm, dm = Mat.out(M, K, 5, 8), Mat(x, 8, 8), Mat(dh, 3, 1)
        need = ghip.apus_ghip_mxfp4_gated_backward_ws(M, N, K)
        ws = Mat.out(1, need // 2)
        ok(ghip, ghip.apus_ghip_mxfp4_gated_backward_dev(G.vp(wg.codes), G.vp(wg.scales), G.vp(wu.codes), G.vp(wu.scales), xm.p, dm.p, dx.p,
                                                         M, N, K, xm.ld, dm.ld, dx.ld, act, limit, ws.p, need, None))
        R.check(wide(dx.get()), *R.gated_backward(wide(x), wg.values, wu.values, wide(dh), act, limit)["dx"], "dx")
        ws.get()


# ---- as they are used ------------------------------------------------------------


def block(lib, M, D, I, b, xt, st=None):
    """Norm, gate and up, quantization between, down onto the stream."""
    vp = G.vp
    codes, scales = (vp(b["c"]), vp(b["cs"])) if xt else (None, None)
    y = None if xt else vp(b["y"])
    ok(lib, lib.apus_ghip_rmsnorm_dev(vp(b["x"]), vp(b["r"]), vp(b["g"]), vp(b["s"]), y, codes, scales, None, M, D, 0, 0, 0, 0, 1e-5, st))
    x = (xt, codes, scales) if xt else (0, y, None)
    ok(lib, lib.apus_ghip_mxfp4_gated_dev(vp(b["wg"].codes), vp(b["wg"].scales), vp(b["wu"].codes), vp(b["wu"].scales), *x, vp(b["h"]), M, I,
                                          D, 0, 0, R.SILU, 10.0, st))
    h = (0, vp(b["h"]), None)
    if xt:
        ok(lib, lib.apus_ghip_mx_quantize_dev(xt, vp(b["h"]), vp(b["hc"]), vp(b["hs"]), M, I, 0, st))
        h = (xt, vp(b["hc"]), vp(b["hs"]))
    ok(lib, lib.apus_ghip_mxfp4_linear_dev(vp(b["wd"].codes), vp(b["wd"].scales), *h, None, vp(b["s"]), vp(b["out"]), M, D, I, 0, 0, 0, R.NONE, st))


@pytest.mark.parametrize("M", [1, 5, 130, 600])
@pytest.mark.parametrize("xt", [X.BF16, X.MXFP8])
def test_a_block_eager_and_replayed(ghip, M, xt):
    """A feed-forward block onto the residual stream: each step against the 64-bit form of what the step before gave, then
    captured and replayed with other inputs between eager runs on another stream."""
    rt, (D, I) = G.rt(), (544, 1056)
    rng = seed(51, M, xt)
    wts = {"wg": weights(rng, I, D, 3.0), "wu": weights(rng, I, D, 3.0), "wd": weights(rng, D, I)}
    gamma = G.dev(bf(1 + 0.1 * rng.standard_normal(D)))

    def buffers(x, r):
        sizes = {"x": 2 * M * D, "r": 2 * M * D, "s": 2 * M * D, "y": 2 * M * D, "out": 2 * M * D, "h": 2 * M * I, "c": M * D,
                 "cs": M * X.scale_ld(D), "hc": M * I, "hs": M * X.scale_ld(I)}
        return {**{k: G.empty(n) for k, n in sizes.items()}, **wts, "g": gamma, "x": x, "r": r}

    x, r = G.empty(2 * M * D), G.empty(2 * M * D)
    x.upload(acts(rng, M, D)), r.upload(bf(rng.standard_normal((M, D))))
    a = buffers(x, r)
    block(ghip, M, D, I, a, xt)
    g16 = lambda k, n: G.host(a[k], np.uint16, (M, n))  # noqa: E731
    s, h, out = g16("s", D), g16("h", I), g16("out", D)
    y, err, _ = X.norm(wide(s), wide(gamma.download(np.uint16, D)), 1e-5)
    if xt:
        c, cs = G.host(a["c"], np.uint8, (M, D)), G.host(a["cs"], np.uint8, (M, X.scale_ld(D)))
        from test_gpu_norm import check_mx
        check_mx(c, cs, y, err)
        xin = X.values(xt, c, cs)
        want = X.quantize(xt, wide(h))
        assert np.array_equal(G.host(a["hc"], np.uint8, (M, I)), want[0]) and np.array_equal(G.host(a["hs"], np.uint8, (M, X.scale_ld(I))), want[1])
        hin = X.values(xt, *want)
    else:
        xin, hin = wide(g16("y", D)), wide(h)
        R.check(xin, y, err + X.HALF * np.abs(y), "norm")
    R.check(wide(h), *X.gated(xin, wts["wg"].values, wts["wu"].values, R.SILU, 10.0, xt), "gated")
    R.check(wide(out), *X.linear(hin, wts["wd"].values, None, wide(s), R.NONE, xt), "down")

    b, st, other = buffers(x, r), rt.Stream(), rt.Stream()
    graph = rt.Graph(st)
    graph.begin()
    block(ghip, M, D, I, a, xt, st.vp)
    graph.end()
    for k in range(4):
        x.upload(acts(seed(52, k), M, D)), r.upload(bf(seed(53, k).standard_normal((M, D))))
        graph.launch()
        block(ghip, M, D, I, b, xt, other.vp)
        st.synchronize()
        other.synchronize()
        for key in ("s", "h", "out"):
            n = a[key].nbytes // 2
            assert np.array_equal(a[key].download(np.uint16, n), b[key].download(np.uint16, n)), key
    graph.close()


def test_a_tuning_step_through_frozen_weights(ghip):
    """Norm, gated, down and back: dx of the stream by the entries in reverse, each against the 64-bit form of what the
    step before gave."""
    M, D, I = 70, 160, 288
    rng = seed(54)
    wg, wu, wd = weights(rng, I, D, 3.0), weights(rng, I, D, 3.0), weights(rng, D, I)
    x, dout, gamma = acts(rng, M, D), bf(rng.standard_normal((M, D))), bf(1 + 0.1 * rng.standard_normal((1, D)))
    y, h, dx = Mat.out(M, D), Mat.out(M, I), Mat.out(M, D)
    xm, gm, om = Mat(x), Mat(gamma), Mat(dout)
    ok(ghip, ghip.apus_ghip_rmsnorm_dev(xm.p, None, gm.p, None, y.p, None, None, None, M, D, 0, 0, 0, 0, 1e-5, None))
    yc = y.get()
    ok(ghip, gated(ghip, wg, wu, Act(X.BF16, yc), h, R.SILU, 2.0))
    dh = run_linear_bwd(ghip, wd, None, None, om, R.NONE, ("dx",))["dx"]
    R.check(wide(dh), *R.linear_backward(wide(h.get()), wd.values, None, wide(dout), R.NONE)["dx"], "dh")
    need = ghip.apus_ghip_mxfp4_gated_backward_ws(M, I, D)
    ws, dyc, hm = G.empty(need), Mat.out(M, D), Mat(dh)
    ok(ghip, ghip.apus_ghip_mxfp4_gated_backward_dev(G.vp(wg.codes), G.vp(wg.scales), G.vp(wu.codes), G.vp(wu.scales), y.p, hm.p, dyc.p,
                                                     M, I, D, 0, 0, 0, R.SILU, 2.0, G.vp(ws), need, None))
    dy = dyc.get()
    R.check(wide(dy), *R.gated_backward(wide(yc), wg.values, wu.values, wide(dh), R.SILU, 2.0)["dx"], "dy")
    need = ghip.apus_ghip_rmsnorm_backward_ws(M, D)
    ws, dg = G.empty(need), Mat.out(1, D)
    ok(ghip, ghip.apus_ghip_rmsnorm_backward_dev(xm.p, gm.p, None, dyc.p, om.p, dx.p, dg.p, M, D, 0, 0, 0, 0, 1e-5, G.vp(ws), need, None))
    wx, wgm = X.norm_backward(wide(x), wide(gamma)[0], wide(dy), wide(dout), 1e-5)
    R.check(wide(dx.get()), *wx, "dx")
    R.check(wide(dg.get())[0], *wgm, "dgamma")


def test_two_streams_at_once(ghip):
    """Products of both routes and the backward passes on two streams at a time, each with its own buffers."""
    rt = G.rt()
    M, N, K = 300, 520, 640
    rng = seed(55)
    w, w2 = weights(rng, N, K), weights(rng, N, K)
    xs = [Act(t, acts(rng, M, K)) for t in XTYPES]
    few = [Act(t, acts(rng, 3, K)) for t in XTYPES]
    sts = [rt.Stream(), rt.Stream()]
    alone = []
    for a in xs + few:
        y = Mat.out(a.values.shape[0], N)
        ok(ghip, gated(ghip, w, w2, a, y, R.SILU, 0.0))
        alone.append(y.get())
    outs = [[Mat.out(a.values.shape[0], N) for a in xs + few] for _ in sts]
    for _ in range(3):
        for k, a in enumerate(xs + few):
            for st, o in zip(sts, outs):
                ok(ghip, gated(ghip, w, w2, a, o[k], R.SILU, 0.0, st.vp))
    for st, o in zip(sts, outs):
        st.synchronize()
        assert all(np.array_equal(y.get(), v) for y, v in zip(o, alone))
