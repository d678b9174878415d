"""The dense feed-forward entries on the device against tests/ffn_ref.py's
64-bit forms: shapes of every route, strides and alignments, clamps and
infinities, gradients left out, streams and graphs."""
import ctypes

import numpy as np
import pytest

import ffn_ref as R
import gpu_util as G
import oracle as O

pytestmark = pytest.mark.gpu

FILL = 0x7E57                                                       # what output buffers hold before a call


def bf(a):
    return O.f32_to_bf16(np.ascontiguousarray(a, np.float32))


def wide(b):
    return O.bf16_to_f32(b).astype(np.float64)


class Mat:
    """A [rows, cols] matrix of bf16 codes on the device: `pad` columns more a
    row, `off` elements into its buffer; the rest holds `fill`."""

    def __init__(self, codes, pad=0, off=0, fill=FILL):
        self.rows, self.cols = codes.shape
        self.ld, self.off = self.cols + pad, off
        host = np.full(off + self.rows * self.ld + 64, fill, np.uint16)
        self.view(host)[:, :self.cols] = codes
        self.before, self.buf = host, G.dev(host)

    def view(self, host):
        return host[self.off:self.off + self.rows * self.ld].reshape(self.rows, self.ld)

    @classmethod
    def out(cls, rows, cols, pad=0, off=0):
        return cls(np.full((rows, cols), FILL, np.uint16), pad, off)

    @property
    def p(self):
        return ctypes.c_void_p(G.vp(self.buf).value + 2 * self.off)

    def get(self):
        """Its values, once nothing around them has changed."""
        host = G.host(self.buf, np.uint16, self.before.shape)
        got, was = self.view(host)[:, :self.cols].copy(), self.before.copy()
        self.view(was)[:, :self.cols] = got
        assert np.array_equal(host, was), "wrote outside the matrix"
        return got


def ok(lib, rc):
    assert rc == 0, lib.apus_ghip_last_error()


def fp8(rng, N, K, nans=False):
    codes = rng.integers(0, 254, (N, K), dtype=np.uint8)
    codes[codes >= 0x7F] += 1
    if nans:
        codes[rng.random((N, K)) < 0.01] = 0x7F
        codes[rng.random((N, K)) < 0.01] = 0xFF
    scales = np.exp2(rng.uniform(-13, -11, ((N + 127) // 128, (K + 127) // 128))).astype(np.float32)
    return codes, scales


def seed(*a):
    return np.random.default_rng([int(v) for v in a])


# M, N, K: one row, a few, tiles and their edges, K of one step and of ragged ends
SHAPES = [(1, 1, 1), (1, 5, 8), (1, 300, 2048), (2, 4096, 128), (3, 257, 100), (4, 1000, 4096), (5, 96, 264), (2, 200, 1080), (9, 77, 24), (1, 40, 8), (7, 2050, 640),
          (8, 129, 1536), (13, 64, 64), (16, 768, 192), (17, 33, 31), (31, 520, 1000), (33, 1025, 576), (64, 512, 1024),
          (65, 255, 72), (100, 2048, 512), (129, 130, 131), (200, 1537, 320), (255, 257, 256), (256, 256, 64), (300, 520, 1088),
          (513, 1032, 136), (700, 2049, 192), (1111, 640, 448), (2049, 1030, 256)]


def data(M, N, K, weights, op, rng, nans=False):
    x = bf(rng.standard_normal((M, K)))
    out = []
    for _ in range(2 if op == "gated" else 1):
        if weights == "fp8":
            codes, scales = fp8(rng, N, K, nans)
            out.append((codes, scales, wide(O.dequant(codes, scales))))
        else:
            w = bf(rng.standard_normal((N, K)) / np.sqrt(K))
            out.append((w, None, wide(w)))
    return x, out


def call_linear(lib, w, x, bias, res, y, M, N, K, act, exact=0, st=None):
    """w: (codes or bf16, scales or None) device buffers; x, res, y: Mat."""
    b = None if bias is None else G.vp(bias)
    r, ldr = (None, 0) if res is None else (res.p, res.ld)
    if w[1] is not None:
        return lib.apus_ghip_fp8blk_linear_ep_dev(G.vp(w[0]), G.vp(w[1]), x.p, b, r, y.p, M, N, K, x.ld, ldr, y.ld, act, exact, st)
    return lib.apus_ghip_bf16_linear_ep_dev(G.vp(w[0]), x.p, b, r, y.p, M, N, K, x.ld, ldr, y.ld, act, st)


def call_gated(lib, wg, wu, x, h, M, N, K, act, limit, exact=0, st=None):
    if wg[1] is not None:
        return lib.apus_ghip_fp8blk_gated_dev(G.vp(wg[0]), G.vp(wg[1]), G.vp(wu[0]), G.vp(wu[1]), x.p, h.p, M, N, K, x.ld, h.ld,
                                              act, limit, exact, st)
    return lib.apus_ghip_bf16_gated_dev(G.vp(wg[0]), G.vp(wu[0]), x.p, h.p, M, N, K, x.ld, h.ld, act, limit, st)


def dev_w(w):
    return G.dev(w[0]), None if w[1] is None else G.dev(w[1])


@pytest.mark.parametrize("weights", ["bf16", "fp8"])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear(ghip, M, N, K, weights):
    i = SHAPES.index((M, N, K))
    rng, act = seed(1, M, N, K), R.ACTS[i % 5]
    bias = bf(rng.standard_normal(N)) if i % 2 else None
    res = bf(rng.standard_normal((M, N))) if i % 3 else None
    x, [w] = data(M, N, K, weights, "linear", rng)
    y = Mat.out(M, N, off=8)
    ok(ghip, call_linear(ghip, dev_w(w), Mat(x), None if bias is None else G.dev(bias), None if res is None else Mat(res), y,
                         M, N, K, act))
    want, tol = R.linear(wide(x), w[2], None if bias is None else wide(bias), None if res is None else wide(res), act)
    R.check(wide(y.get()), want, tol, "linear")


@pytest.mark.parametrize("weights", ["bf16", "fp8"])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_gated(ghip, M, N, K, weights):
    i = SHAPES.index((M, N, K))
    act, limit = R.ACTS[(i + 2) % 5], (0.0, 1.5)[i % 2]
    x, [wg, wu] = data(M, N, K, weights, "gated", seed(2, M, N, K))
    h = Mat.out(M, N, off=8)
    ok(ghip, call_gated(ghip, dev_w(wg), dev_w(wu), Mat(x), h, M, N, K, act, limit))
    want, tol = R.gated(wide(x), wg[2], wu[2], act, limit)
    R.check(wide(h.get()), want, tol, "gated")


def run_linear_bwd(lib, w, x, bias, dy, M, N, K, act, want=("dx", "dw", "db"), st=None, pad=0):
    out = {"dx": Mat.out(M, K, pad, 8), "dw": Mat.out(N, K, 0, 8), "db": Mat.out(1, N, 0, 8)}
    need = lib.apus_ghip_linear_ep_backward_ws(M, N, K)
    ws = Mat.out(1, need // 2)
    p = lambda k: out[k].p if k in want else None  # noqa: E731
    ok(lib, lib.apus_ghip_bf16_linear_ep_backward_dev(
        G.vp(w), x.p, None if bias is None else G.vp(bias), dy.p, p("dx"), p("dw"), p("db"), M, N, K, x.ld, dy.ld, out["dx"].ld,
        act, ws.p, need, st))
    got = {k: m.get() for k, m in out.items()}
    ws.get()                                                        # nothing past the workspace
    return got


def run_gated_bwd(lib, wg, wu, x, dh, M, N, K, act, limit, want=("dx", "dwg", "dwu"), st=None, pad=0):
    out = {"dx": Mat.out(M, K, pad, 8), "dwg": Mat.out(N, K, 0, 8), "dwu": Mat.out(N, K, 0, 8)}
    need = lib.apus_ghip_gated_backward_ws(M, N, K)
    ws = Mat.out(1, need // 2)
    p = lambda k: out[k].p if k in want else None  # noqa: E731
    ok(lib, lib.apus_ghip_bf16_gated_backward_dev(
        G.vp(wg), G.vp(wu), x.p, dh.p, p("dx"), p("dwg"), p("dwu"), M, N, K, x.ld, dh.ld, out["dx"].ld, act, limit, ws.p, need,
        st))
    got = {k: m.get() for k, m in out.items()}
    ws.get()
    return got


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear_backward(ghip, M, N, K):
    i = SHAPES.index((M, N, K))
    rng, act = seed(3, M, N, K), R.ACTS[(i // 2) % 5]
    x, [w] = data(M, N, K, "bf16", "linear", rng)
    bias, dy = bf(rng.standard_normal(N)) if i % 2 else None, bf(rng.standard_normal((M, N)))
    got = run_linear_bwd(ghip, G.dev(w[0]), Mat(x), None if bias is None else G.dev(bias), Mat(dy), M, N, K, act)
    want = R.linear_backward(wide(x), w[2], None if bias is None else wide(bias), wide(dy), act)
    for k, v in (("dx", "dx"), ("dw", "dw0")):
        R.check(wide(got[k]), *want[v], k)
    R.check(wide(got["db"])[0], *want["db"], "db")


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_gated_backward(ghip, M, N, K):
    i = SHAPES.index((M, N, K))
    act, limit = R.ACTS[(i + 2) % 5], (1.5, 0.0)[i % 2]
    rng = seed(4, M, N, K)
    x, [wg, wu] = data(M, N, K, "bf16", "gated", rng)
    dh = bf(rng.standard_normal((M, N)))
    got = run_gated_bwd(ghip, G.dev(wg[0]), G.dev(wu[0]), Mat(x), Mat(dh), M, N, K, act, limit)
    want = R.gated_backward(wide(x), wg[2], wu[2], wide(dh), act, limit)
    for k, v in (("dx", "dx"), ("dwg", "dw0"), ("dwu", "dw1")):
        R.check(wide(got[k]), *want[v], k)


@pytest.mark.parametrize("weights", ["bf16", "fp8"])
@pytest.mark.parametrize("M,N,K", [(1, 520, 512), (6, 264, 256), (40, 392, 384), (40, 392, 208), (300, 520, 640), (300, 520, 1104)])
@pytest.mark.parametrize("pad,off", [(8, 8), (64, 0), (3, 1), (1, 0), (8, 3)])
def test_rows_in_wider_buffers(ghip, M, N, K, weights, pad, off):
    """x, residual and y as slices of wider buffers, 16-byte aligned or not: the
    same values bit for bit or within the tolerance, nothing else written (the
    rest of x's buffer holds NaN codes)."""
    rng = seed(5, M, N, K)
    x, [w, w2] = data(M, N, K, weights, "gated", rng)
    res = bf(rng.standard_normal((M, N)))
    y, h = Mat.out(M, N, pad, off), Mat.out(M, N, pad, off)
    xd = Mat(x, pad, off, 0x7FC0)
    ok(ghip, call_linear(ghip, dev_w(w), xd, None, Mat(res, pad, off, 0x7FC0), y, M, N, K, R.NONE))
    R.check(wide(y.get()), *R.linear(wide(x), w[2], None, wide(res), R.NONE), "linear")
    ok(ghip, call_gated(ghip, dev_w(w), dev_w(w2), xd, h, M, N, K, R.SILU, 2.0))
    R.check(wide(h.get()), *R.gated(wide(x), w[2], w2[2], R.SILU, 2.0), "gated")


@pytest.mark.parametrize("M,N,K", [(6, 264, 256), (300, 520, 640), (300, 515, 200)])
@pytest.mark.parametrize("pad,off", [(8, 8), (3, 1)])
def test_backward_of_rows_in_wider_buffers(ghip, M, N, K, pad, off):
    rng = seed(6, M, N, K)
    x, [w, w2] = data(M, N, K, "bf16", "gated", rng)
    dy = bf(rng.standard_normal((M, N)))
    xd, dd = Mat(x, pad, off, 0x7FC0), Mat(dy, pad, off, 0x7FC0)
    got = run_linear_bwd(ghip, G.dev(w[0]), xd, None, dd, M, N, K, R.GELU, pad=pad)
    want = R.linear_backward(wide(x), w[2], None, wide(dy), R.GELU)
    R.check(wide(got["dx"]), *want["dx"], "dx")
    R.check(wide(got["dw"]), *want["dw0"], "dw")
    got = run_gated_bwd(ghip, G.dev(w[0]), G.dev(w2[0]), xd, dd, M, N, K, R.SILU, 2.0, pad=pad)
    want = R.gated_backward(wide(x), w[2], w2[2], wide(dy), R.SILU, 2.0)
    for k, v in (("dx", "dx"), ("dwg", "dw0"), ("dwu", "dw1")):
        R.check(wide(got[k]), *want[v], k)


@pytest.mark.parametrize("M,N,K", [(1, 4096, 1024), (9, 1040, 512), (333, 777, 192)])
def test_residual_in_place(ghip, M, N, K):
    """y += act(x W^T): the residual's own buffer as the output."""
    rng = seed(7, M, N, K)
    x, [w] = data(M, N, K, "bf16", "linear", rng)
    res = bf(rng.standard_normal((M, N)))
    y, other = Mat(res, 8, 8), Mat.out(M, N)
    ok(ghip, call_linear(ghip, dev_w(w), Mat(x), None, y, y, M, N, K, R.GELU))
    ok(ghip, call_linear(ghip, dev_w(w), Mat(x), None, Mat(res), other, M, N, K, R.GELU))
    got = y.get()
    R.check(wide(got), *R.linear(wide(x), w[2], None, wide(res), R.GELU), "in place")
    assert np.array_equal(got, other.get())


@pytest.mark.parametrize("M,N,K", [(1, 512, 512), (5, 136, 256), (40, 392, 384), (270, 264, 512), (270, 264, 200)])
def test_nan_codes(ghip, M, N, K):
    """exact != 0 (and -1): codes 0x7F and 0xFF decode as +-480."""
    x, [w, w2] = data(M, N, K, "fp8", "gated", seed(8, M, N, K), nans=True)
    for exact in (1, -1):
        y, h = Mat.out(M, N), Mat.out(M, N)
        ok(ghip, call_linear(ghip, dev_w(w), Mat(x), None, None, y, M, N, K, R.NONE, exact))
        R.check(wide(y.get()), *R.linear(wide(x), w[2], None, None, R.NONE), "linear")
        ok(ghip, call_gated(ghip, dev_w(w), dev_w(w2), Mat(x), h, M, N, K, R.SILU, 0.0, exact))
        R.check(wide(h.get()), *R.gated(wide(x), w[2], w2[2], R.SILU, 0.0), "gated")


@pytest.mark.parametrize("M", [3, 70, 300])
@pytest.mark.parametrize("K", [128, 136])
def test_not_finite_values_stay_in_their_rows(ghip, M, K):
    """An infinity in x's last row and a NaN in w's last row reach exactly their
    own row and column (rows and columns past the edge are never read into
    another's result); a residual's infinity its own element."""
    N = 265
    rng = seed(9, M)
    w, x = rng.uniform(1, 2, (N, K)), rng.uniform(1, 2, (M, K))
    w, x, res = bf(w), bf(x), bf(rng.standard_normal((M, N)))
    x[M - 1, K - 1], w[N - 1, 7], res[1, 2] = 0x7F80, 0x7FC0, 0xFF80
    for off in (0, 1):
        y = Mat.out(M, N, 0, off)
        ok(ghip, call_linear(ghip, (G.dev(w), None), Mat(x, 0, off), None, Mat(res, 0, off), y, M, N, K, R.NONE))
        got = O.bf16_to_f32(y.get())
        assert np.all(np.isnan(got[:, N - 1])) and np.all(np.isposinf(got[M - 1, :N - 1])) and np.isneginf(got[1, 2])
        got[1, 2] = 0
        assert np.all(np.isfinite(got[:M - 1, :N - 1]))


@pytest.mark.parametrize("M", [2, 50, 300])
def test_clamps_of_infinite_sums(ghip, M):
    """Gates and ups far past the limit, infinite ones among them: h is
    act(limit) * +-limit, and no gradient (not 0 * inf) passes the clamp."""
    N, K, limit = 72, 64, 10.0
    rng = seed(10, M)
    x = np.zeros((M, K))
    x[:, 0] = 1
    wg, wu = np.zeros((N, K)), np.zeros((N, K))
    wg[:, 0] = np.where(np.arange(N) % 3 == 0, 3e38, 50.0)
    wu[:, 0] = np.where(np.arange(N) % 2, 3e38, -70.0)
    x[0, 0] = 3e38                                                  # sums of +-inf
    dh = bf(rng.standard_normal((M, N)))
    dh[0, 0] = 0x7F80
    xd, g, u = bf(x), bf(wg), bf(wu)
    h = Mat.out(M, N)
    ok(ghip, call_gated(ghip, (G.dev(g), None), (G.dev(u), None), Mat(xd), h, M, N, K, R.SILU, limit))
    a = 10.0 / (1 + np.exp(-10.0))
    want = np.broadcast_to(np.where(np.arange(N) % 2, a * limit, -a * limit), (M, N))
    R.check(wide(h.get()), want, HALF2 * np.abs(want), "h")
    got = run_gated_bwd(ghip, G.dev(g), G.dev(u), Mat(xd), Mat(dh), M, N, K, R.SILU, limit)
    assert all(not np.any(v & 0x7FFF) for v in got.values())


HALF2 = 2.0 ** -8 + 2.0 ** -20


def test_an_activation_of_far_sums(ghip):
    """act and its slope at sums of 0, tiny, large and infinite magnitude, each
    passed through a weight of 1: finite where the 64-bit form is, and equal to
    a step."""
    z = np.concatenate([np.linspace(-120, 120, 4001), [0.0, -0.0, 1e-30, -1e-30, 1e30, -1e30]])
    z = wide(bf(z))
    M, N, K = len(z), 8, 64
    x = np.zeros((M, K), np.float32)
    x[:, 0] = z
    w = np.zeros((N, K), np.float32)
    w[:, 0] = 1
    one = bf(np.ones((M, N)))
    for a in R.ACTS:
        y = Mat.out(M, N)
        ok(ghip, call_linear(ghip, (G.dev(bf(w)), None), Mat(bf(x)), None, None, y, M, N, K, a))
        with np.errstate(over="ignore", invalid="ignore"):
            want = np.nan_to_num(R.act(a, z))
        tol = R._eval(z) + R.HALF * np.abs(want) + 1e-37
        R.check(wide(y.get()), np.repeat(want[:, None], N, 1), np.repeat(tol[:, None], N, 1), "act %d" % a)
        # dx of one column that dy selects: act'(z)
        dy = np.zeros((M, N), np.uint16)
        dy[:, 3] = one[:, 3]
        got = run_linear_bwd(ghip, G.dev(bf(w)), Mat(bf(x)), None, Mat(dy), M, N, K, a, want=("dx",))["dx"]
        s = R.slope(a, np.clip(z, -100, 100))
        R.check(wide(got)[:, 0], s, R._eval(np.clip(z, -100, 100)) + 2 * HALF2 * np.abs(s) + 1e-37, "slope %d" % a)


def test_gradients_left_out(ghip):
    """A NULL gradient is not computed and changes no other one."""
    M, N, K = 90, 200, 136
    rng = seed(11)
    x, [w, w2] = data(M, N, K, "bf16", "gated", rng)
    dy = Mat(bf(rng.standard_normal((M, N))))
    xd, a, b = Mat(x), G.dev(w[0]), G.dev(w2[0])
    full = run_linear_bwd(ghip, a, xd, None, dy, M, N, K, R.SILU)
    none = run_linear_bwd(ghip, a, xd, None, dy, M, N, K, R.NONE)
    for k in full:
        assert np.array_equal(run_linear_bwd(ghip, a, xd, None, dy, M, N, K, R.SILU, want=(k,))[k], full[k])
        assert np.array_equal(run_linear_bwd(ghip, a, xd, None, dy, M, N, K, R.NONE, want=(k,))[k], none[k])
    full = run_gated_bwd(ghip, a, b, xd, dy, M, N, K, R.SILU, 2.0)
    for k in full:
        part = run_gated_bwd(ghip, a, b, xd, dy, M, N, K, R.SILU, 2.0, want=(k,))
        assert np.array_equal(part[k], full[k])
        assert all(np.all(part[o] == FILL) for o in full if o != k)


BLOCKS = [(1, 1024, 512, "fp8"), (5, 512, 384, "bf16"), (77, 520, 264, "bf16"), (260, 768, 512, "fp8")]


def block(M, I, D, weights):
    """A feed-forward block: y = x + down(gated(x))."""
    rng = seed(12, M, I, D)
    x, [wg, wu] = data(M, I, D, weights, "gated", rng)
    _, [wd] = data(1, D, I, weights, "linear", rng)
    return x, wg, wu, wd


@pytest.mark.parametrize("M,I,D,weights", BLOCKS)
def test_a_block(ghip, M, I, D, weights):
    """gated, then the down projection onto the residual stream, in place."""
    x, wg, wu, wd = block(M, I, D, weights)
    h, y, xd = Mat.out(M, I), Mat(x, 8), Mat(x)
    g, u, d = dev_w(wg), dev_w(wu), dev_w(wd)
    ok(ghip, call_gated(ghip, g, u, xd, h, M, I, D, R.SILU, 10.0))
    ok(ghip, call_linear(ghip, d, h, None, y, y, M, D, I, R.NONE))
    hv, ht = R.gated(wide(x), wg[2], wu[2], R.SILU, 10.0)
    yv, yt = R.linear(hv, wd[2], None, wide(x), R.NONE)
    R.check(wide(y.get()), yv, yt + ht @ np.abs(wd[2]).T * 1.01, "block")


@pytest.mark.parametrize("M,I,D", [(40, 264, 128), (300, 520, 256)])
def test_a_training_step(ghip, M, I, D):
    """The block's gradients through both backward passes: dh from the down
    projection's, then the gated one's, and dx of the residual beside it."""
    x, wg, wu, wd = block(M, I, D, "bf16")
    rng = seed(13)
    dy = bf(rng.standard_normal((M, D)))
    xd, g, u, d, h = Mat(x), dev_w(wg), dev_w(wu), dev_w(wd), Mat.out(M, I)
    ok(ghip, call_gated(ghip, g, u, xd, h, M, I, D, R.SILU, 10.0))
    down = run_linear_bwd(ghip, d[0], h, None, Mat(dy), M, D, I, R.NONE)
    got = run_gated_bwd(ghip, g[0], u[0], xd, Mat(down["dx"]), M, I, D, R.SILU, 10.0)
    hv, ht = R.gated(wide(x), wg[2], wu[2], R.SILU, 10.0)
    dh = wide(dy) @ wd[2]
    want = R.gated_backward(wide(x), wg[2], wu[2], dh, R.SILU, 10.0)
    # dh's rounding, dg's and du's, the output's: three half steps
    for k, v in (("dx", "dx"), ("dwg", "dw0"), ("dwu", "dw1")):
        n = np.linalg.norm(want[v][0])
        assert np.linalg.norm(wide(got[k]) - want[v][0]) <= 3 * R.HALF / np.sqrt(3) * n, k
    dw = wide(dy).T @ hv
    assert np.linalg.norm(wide(down["dw"]) - dw) <= 2 * R.HALF / np.sqrt(3) * np.linalg.norm(dw)


def test_deterministic(ghip):
    """The same bits twice, forward and backward."""
    for M in (1, 30, 300):
        N, K = 520, 1032
        rng = seed(14, M)
        x, [w, w2] = data(M, N, K, "bf16", "gated", rng)
        dy, xd, a, b = Mat(bf(rng.standard_normal((M, N)))), Mat(x), G.dev(w[0]), G.dev(w2[0])
        runs = [run_gated_bwd(ghip, a, b, xd, dy, M, N, K, R.SILU, 2.0) for _ in range(2)]
        assert all(np.array_equal(runs[0][k], runs[1][k]) for k in runs[0])
        hs = []
        for _ in range(2):
            h = Mat.out(M, N)
            ok(ghip, call_gated(ghip, (a, None), (b, None), xd, h, M, N, K, R.SILU, 2.0))
            hs.append(h.get())
        assert np.array_equal(*hs)


@pytest.mark.parametrize("M,I,D,weights", BLOCKS)
def test_two_streams_and_graphs(ghip, M, I, D, weights):
    """A block captured on each of two streams; both graphs replayed several
    times at once, with eager calls between: every replay gives the eager bits."""
    rt = G.rt()
    cases = []
    for k in range(2):
        x, wg, wu, wd = block(M + k, I, D, weights)
        h, y, xd = Mat.out(M + k, I), Mat.out(M + k, D), Mat(x)
        g, u, d = dev_w(wg), dev_w(wu), dev_w(wd)

        def call(st, h=h, y=y, xd=xd, g=g, u=u, d=d, m=M + k):
            ok(ghip, call_gated(ghip, g, u, xd, h, m, I, D, R.SILU, 10.0, st=st))
            ok(ghip, call_linear(ghip, d, h, None, xd, y, m, D, I, R.NONE, st=st))
        call(None)
        cases.append((call, h, y, h.get(), y.get()))
    graphs = []
    for call, *_ in cases:
        st = rt.Stream()
        gr = rt.Graph(st)
        gr.begin()
        call(st.vp)
        gr.end()
        graphs.append(gr)
    blank = [[np.full(m.before.shape, FILL, np.uint16) for m in c[1:3]] for c in cases]
    for _ in range(3):
        for (_, h, y, _, _), b in zip(cases, blank):
            h.buf.upload(b[0])
            y.buf.upload(b[1])
        for gr in graphs:
            gr.launch()
        for gr in graphs:
            gr.stream.synchronize()
        for _, h, y, hw, yw in cases:
            assert np.array_equal(h.get(), hw) and np.array_equal(y.get(), yw)
        cases[0][0](None)                                           # eager work between the replays
        rt.synchronize()
    for gr in graphs:
        gr.close()


def test_backward_graphs(ghip):
    """A captured backward pass, replayed while another one with a workspace of
    its own runs on a second stream."""
    rt = G.rt()
    M, N, K = 130, 264, 192
    cases = []
    for k in range(2):
        rng = seed(15, k)
        x, [w, w2] = data(M, N, K, "bf16", "gated", rng)
        xd, dd, a, b = Mat(x), Mat(bf(rng.standard_normal((M, N)))), G.dev(w[0]), G.dev(w2[0])
        out, need = [Mat.out(M, K), Mat.out(N, K), Mat.out(N, K)], ghip.apus_ghip_gated_backward_ws(M, N, K)
        ws, st = Mat.out(1, need // 2), rt.Stream()
        want = run_gated_bwd(ghip, a, b, xd, dd, M, N, K, R.SILU, 2.0)
        gr = rt.Graph(st)
        gr.begin()
        ok(ghip, ghip.apus_ghip_bf16_gated_backward_dev(G.vp(a), G.vp(b), xd.p, dd.p, *[o.p for o in out], M, N, K, 0, 0, 0,
                                                         R.SILU, 2.0, ws.p, need, st.vp))
        gr.end()
        cases.append((gr, out, [want[n] for n in ("dx", "dwg", "dwu")], (xd, dd, a, b, ws)))
    for _ in range(3):
        for _, out, _, _ in cases:
            for o in out:
                o.buf.upload(o.before)
        for gr, *_ in cases:
            gr.launch()
        for gr, *_ in cases:
            gr.stream.synchronize()
        for _, out, want, _ in cases:
            assert all(np.array_equal(o.get(), v) for o, v in zip(out, want))
    for gr, *_ in cases:
        gr.close()


def test_rows_far_apart(ghip):
    """Rows of x, residual and y 2^30 elements apart: offsets past 32 bits."""
    rt = G.rt()
    M, N, K, ld = 3, 200, 256, 1 << 30
    free, _ = rt.mem_info()
    need = 2 * ((M - 1) * ld + 512)
    if free < 3 * need:
        pytest.skip("needs %d GiB of device memory" % (3 * need >> 30))
    rng = seed(16)
    x, [w, w2] = data(M, N, K, "bf16", "gated", rng)
    res = bf(rng.standard_normal((M, N)))
    bufs = [G.empty(need) for _ in range(3)]
    base = [G.vp(b).value for b in bufs]

    def put(at, rows):
        for m in range(M):
            r = np.ascontiguousarray(rows[m])
            rt.check(rt.hip().hipMemcpy(ctypes.c_void_p(at + 2 * m * ld), r.ctypes.data_as(ctypes.c_void_p), r.nbytes, rt.H2D), "copy")

    def take(at, n):
        return np.stack([G.download_ptr(at + 2 * m * ld, np.uint16, (n,)) for m in range(M)])
    put(base[0], x)
    put(base[1], res)
    a, b = G.dev(w[0]), G.dev(w2[0])
    px, pr, py = (ctypes.c_void_p(v) for v in base)
    ok(ghip, ghip.apus_ghip_bf16_linear_ep_dev(G.vp(a), px, None, pr, py, M, N, K, ld, ld, ld, R.NONE, None))
    R.check(wide(take(base[2], N)), *R.linear(wide(x), w[2], None, wide(res), R.NONE), "linear")
    ok(ghip, ghip.apus_ghip_bf16_gated_dev(G.vp(a), G.vp(b), px, py, M, N, K, ld, ld, R.SILU, 0.0, None))
    R.check(wide(take(base[2], N)), *R.gated(wide(x), w[2], w2[2], R.SILU, 0.0), "gated")
    # dh = res, dx over y's buffer
    n = ghip.apus_ghip_gated_backward_ws(M, N, K)
    ws, g1, g2 = G.empty(n), Mat.out(N, K), Mat.out(N, K)
    ok(ghip, ghip.apus_ghip_bf16_gated_backward_dev(G.vp(a), G.vp(b), px, pr, py, g1.p, g2.p, M, N, K, ld, ld, ld, R.SILU, 0.0,
                                                     G.vp(ws), n, None))
    want = R.gated_backward(wide(x), w[2], w2[2], wide(res), R.SILU, 0.0)
    R.check(wide(take(base[2], K)), *want["dx"], "dx")
    R.check(wide(g1.get()), *want["dw0"], "dwg")
    R.check(wide(g2.get()), *want["dw1"], "dwu")
    for v in bufs:
        v.close()
