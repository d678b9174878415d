"""The norm and its gradient on the device against tests/mx_ref.py's 64-bit
forms: rows of every form, strides and alignments, buffers in place, extreme
rows, streams and graphs."""
import numpy as np
import pytest

import ffn_ref as R
import gpu_util as G
import mx_ref as X
import oracle as O
from test_gpu_ffn import Mat, bf, ok, seed, wide

pytestmark = pytest.mark.gpu

EPS = 1e-5
# rows of one element, of a part of a vector, of every form's shortest and longest, of two passes; few rows and more than the
# gradient has blocks
SHAPES = [(1, 1), (1, 7), (1, 8), (1, 4096), (2, 33), (3, 64), (5, 100), (2, 512), (4, 513), (9, 1000), (7, 1024), (6, 1025), (11, 2048),
          (5, 2049), (300, 1536), (33, 4096), (3, 4097), (2, 8192), (4, 8200), (2, 16384), (3, 16385), (2, 40001), (2500, 96),
          (2049, 520), (700, 2056), (1100, 5000)]


class Bytes(Mat):
    """Bytes with 64 more behind them that have to stay."""

    def __init__(self, rows, cols):
        assert rows * cols % 2 == 0
        super().__init__(np.full((1, rows * cols // 2), 0x7E57, np.uint16))
        self.shape = rows, cols

    def get(self):
        return super().get().view(np.uint8).reshape(self.shape)


def f32s(n):
    return Mat(np.zeros((1, 2 * n), np.uint16))


def get_f32(m):
    return m.get().view(np.float32)[0]


def call(lib, x, res, gamma, out, M, D, eps=EPS, st=None):
    p = lambda k: out[k].p if out.get(k) is not None else None  # noqa: E731
    ld = lambda m: 0 if m is None else m.ld  # noqa: E731
    return lib.apus_ghip_rmsnorm_dev(x.p, None if res is None else res.p, None if gamma is None else gamma.p, p("sum"), p("y"), p("codes"),
                                     p("scales"), p("rstd"), M, D, x.ld, ld(res), ld(out.get("sum")), ld(out.get("y")), eps, st)


def inputs(M, D, *tag):
    rng = seed(31, M, D, *tag)
    loud = 1 + 9 * (rng.random(D) < 0.05)
    return (bf(rng.standard_normal((M, D)) * loud), bf(rng.standard_normal((M, D))), bf(1 + 0.3 * rng.standard_normal((1, D))),
            bf(rng.standard_normal((M, D))))


def add(x, r):
    return bf(O.bf16_to_f32(x) + O.bf16_to_f32(r))


def check_mx(codes, scales, y, err):
    """Codes and scales of values that are within err of y: the least scales, to the error, and the nearest codes."""
    M, D = y.shape
    v = X.values(X.MXFP8, codes, scales)
    f = np.exp2(scales[:, :D // 32].astype(float) - 127)
    top, e = np.abs(y).reshape(M, -1, 32).max(2), err.reshape(M, -1, 32).max(2)
    assert np.all(top - e <= 448 * f) and np.all((top + e > 224 * f) | (scales[:, :D // 32] == 0))
    assert not scales[:, D // 32:].any()
    tol = err + 2.0 ** -4 * (np.abs(y) + err) + 2.0 ** -10 * np.repeat(f, 32, 1)
    assert np.all(np.abs(v - y) <= tol)


@pytest.mark.parametrize("M,D", SHAPES)
@pytest.mark.parametrize("residual", [False, True])
def test_norm(ghip, M, D, residual):
    x, r, g, _ = inputs(M, D)
    gain = SHAPES.index((M, D)) % 4 != 1
    s = add(x, r) if residual else x
    out = {"y": Mat.out(M, D, off=8), "rstd": f32s(M)}
    if residual:
        out["sum"] = Mat.out(M, D)
    if D % 32 == 0:
        out |= {"codes": Bytes(M, D), "scales": Bytes(M, X.scale_ld(D))}
    ok(ghip, call(ghip, Mat(x), Mat(r) if residual else None, Mat(g) if gain else None, out, M, D))
    y, err, rstd = X.norm(wide(s), wide(g)[0] if gain else None, EPS)
    if residual:
        assert np.array_equal(out["sum"].get(), s)
    R.check(wide(out["y"].get()), y, err + X.HALF * np.abs(y), "y")
    assert np.all(np.abs(get_f32(out["rstd"]) - rstd) <= ((D + 8) / 2 + 6) * X.U * rstd)
    if D % 32 == 0:
        check_mx(out["codes"].get(), out["scales"].get(), y, err)


@pytest.mark.parametrize("M,D", [(3, 64), (2, 1024), (5, 2048), (300, 4096), (2, 20000 // 32 * 32)])
def test_mxfp8_alone(ghip, M, D):
    """Without y: the same codes as with it."""
    x, r, g, _ = inputs(M, D, 1)
    got = []
    for y in (False, True):
        out = {"codes": Bytes(M, D), "scales": Bytes(M, X.scale_ld(D))}
        if y:
            out["y"] = Mat.out(M, D)
        ok(ghip, call(ghip, Mat(x), Mat(r), Mat(g), out, M, D))
        got.append((out["codes"].get(), out["scales"].get()))
    assert np.array_equal(got[0][0], got[1][0]) and np.array_equal(got[0][1], got[1][1])


@pytest.mark.parametrize("M,D", [(5, 100), (3, 1000), (70, 2048), (4, 4097), (2, 17000)])
@pytest.mark.parametrize("pad,off", [(8, 8), (3, 1), (1, 0)])
def test_rows_in_wider_buffers(ghip, M, D, pad, off):
    x, r, g, dy = inputs(M, D, 2)
    nan = 0x7FC0
    out = {"y": Mat.out(M, D, pad, off), "sum": Mat.out(M, D, pad, off)}
    ok(ghip, call(ghip, Mat(x, pad, off, nan), Mat(r, pad, off, nan), Mat(g, 0, off), out, M, D))
    s = add(x, r)
    assert np.array_equal(out["sum"].get(), s)
    y, err, _ = X.norm(wide(s), wide(g)[0], EPS)
    R.check(wide(out["y"].get()), y, err + X.HALF * np.abs(y), "y")
    got = run_grad(ghip, Mat(s, pad, off, nan), Mat(g, 0, off), None, Mat(dy, pad, off, nan), Mat(r, pad, off, nan), M, D, pad=pad, off=off)
    check_grad(got, s, g, dy, r)


def run_grad(lib, s, gamma, rstd, dy, ds, M, D, want=("dx", "dgamma"), eps=EPS, st=None, pad=0, off=0, dx=None):
    out = {"dx": Mat.out(M, D, pad, off) if dx is None else dx, "dgamma": Mat.out(1, D, 0, off)}
    need = lib.apus_ghip_rmsnorm_backward_ws(M, D)
    ws = Mat.out(1, need // 2)
    p = lambda k: out[k].p if k in want else None  # noqa: E731
    ok(lib, lib.apus_ghip_rmsnorm_backward_dev(s.p, None if gamma is None else gamma.p, None if rstd is None else G.vp(rstd), dy.p,
                                               None if ds is None else ds.p, p("dx"), p("dgamma"), M, D, s.ld, dy.ld,
                                               0 if ds is None else ds.ld, out["dx"].ld, eps, ws.p, need, st))
    got = {k: m.get() for k, m in out.items()}
    ws.get()                                                        # nothing past the workspace
    return got


def check_grad(got, s, g, dy, ds, want=("dx", "dgamma")):
    dx, dg = X.norm_backward(wide(s), None if g is None else wide(g)[0], wide(dy), None if ds is None else wide(ds), EPS)
    if "dx" in want:
        R.check(wide(got["dx"]), *dx, "dx")
    if "dgamma" in want:
        R.check(wide(got["dgamma"])[0], *dg, "dgamma")


@pytest.mark.parametrize("M,D", SHAPES)
@pytest.mark.parametrize("given", [False, True])
def test_gradient(ghip, M, D, given):
    """given: rstd as the norm wrote it."""
    i = SHAPES.index((M, D))
    s, ds, g, dy = inputs(M, D, 3)
    gain, ds = (g if i % 4 != 2 else None), (ds if (i + given) % 2 else None)
    rstd = G.dev((1 / np.sqrt((wide(s) ** 2).mean(1) + EPS)).astype(np.float32)) if given else None
    got = run_grad(ghip, Mat(s), None if gain is None else Mat(gain), rstd, Mat(dy), None if ds is None else Mat(ds), M, D)
    check_grad(got, s, gain, dy, ds)


@pytest.mark.parametrize("M,D", [(13, 96), (13, 2048), (13, 8000), (13, 17024)])
@pytest.mark.parametrize("given", [False, True])
def test_gradient_of_rows_of_any_size(ghip, M, D, given):
    """Rows from 2^-55 to 2^53, whose rstd^3 is no f32."""
    s, _, g, dy = inputs(M, D, 9)
    s = bf(O.bf16_to_f32(s) * np.exp2(np.linspace(-55, 53, M)).astype(np.float32)[:, None])
    rstd = G.dev((1 / np.sqrt((wide(s) ** 2).mean(1))).astype(np.float32)) if given else None
    got = run_grad(ghip, Mat(s), Mat(g), rstd, Mat(dy), None, M, D, eps=0.0)
    dx, dg = X.norm_backward(wide(s), wide(g)[0], wide(dy), None, 0.0)
    for m in range(M):
        R.check(wide(got["dx"])[m:m + 1], dx[0][m:m + 1], dx[1][m:m + 1], "dx %d" % m)
    R.check(wide(got["dgamma"])[0], *dg, "dgamma")


@pytest.mark.parametrize("M,D", [(40, 96), (600, 2048), (3, 5000), (2, 16500)])
def test_gradients_left_out(ghip, M, D):
    s, ds, g, dy = inputs(M, D, 4)
    both = run_grad(ghip, Mat(s), Mat(g), None, Mat(dy), Mat(ds), M, D)
    for want in ("dx", "dgamma"):
        one = run_grad(ghip, Mat(s), Mat(g), None, Mat(dy), Mat(ds), M, D, (want,))
        assert np.array_equal(one[want], both[want])
        other = "dgamma" if want == "dx" else "dx"
        assert np.all(one[other] == 0x7E57)


@pytest.mark.parametrize("M,D", [(5, 100), (300, 1536), (2, 8192), (3, 16385)])
def test_in_place(ghip, M, D):
    """The sum in x's or the residual's buffer, y in the other one; dx in dy's or ds's."""
    x, r, g, dy = inputs(M, D, 5)
    plain = {"y": Mat.out(M, D), "sum": Mat.out(M, D)}
    ok(ghip, call(ghip, Mat(x), Mat(r), Mat(g), plain, M, D))
    want = {k: m.get() for k, m in plain.items()}
    for swap in (False, True):
        a, b = Mat(x, 3), Mat(r, 5)
        out = {"sum": b, "y": a} if swap else {"sum": a, "y": b}
        ok(ghip, call(ghip, a, b, Mat(g), out, M, D))
        assert np.array_equal(out["sum"].get(), want["sum"]) and np.array_equal(out["y"].get(), want["y"])
    grads = run_grad(ghip, Mat(x), Mat(g), None, Mat(dy), Mat(r), M, D)
    for k in range(2):
        d, e = Mat(dy, 1), Mat(r, 2)
        got = run_grad(ghip, Mat(x), Mat(g), None, d, e, M, D, dx=(d, e)[k])
        assert np.array_equal(got["dx"], grads["dx"]) and np.array_equal(got["dgamma"], grads["dgamma"])


@pytest.mark.parametrize("M,D", [(1, 33), (5, 100), (300, 1536), (1024, 520), (1025, 520), (1024, 8192), (600, 9000), (1000, 9000), (130, 16384)])
@pytest.mark.parametrize("place", ["dy", "ds", "own", "none"])
def test_rstd_given(ghip, M, D, place):
    """Few rows and more, dx in dy's buffer, in ds's, in its own and left out."""
    s, ds, g, dy = inputs(M, D, 10)
    rstd = G.dev((1 / np.sqrt((wide(s) ** 2).mean(1) + EPS)).astype(np.float32))
    d, e = Mat(dy, 1), Mat(ds, 2)
    want = ("dgamma",) if place == "none" else ("dx", "dgamma")
    got = run_grad(ghip, Mat(s), Mat(g), rstd, d, e, M, D, want, dx={"dy": d, "ds": e}.get(place))
    check_grad(got, s, g, dy, ds, want)


@pytest.mark.parametrize("D", [96, 1024, 4096, 17024])
def test_extreme_rows(ghip, D):
    """A row of zeros, of the least numbers, of large ones, one with an infinity, one with a NaN: each by the formula, none
    in another's result."""
    M = 6
    x = np.ones((M, D), np.float32)
    x[1], x[2], x[3] = 0, 1e-39, 1e15
    x = bf(x)
    x[4, D - 1], x[5, 3] = 0x7F80, 0x7FC0
    out = {"y": Mat.out(M, D), "codes": Bytes(M, D), "scales": Bytes(M, X.scale_ld(D)), "rstd": f32s(M)}
    ok(ghip, call(ghip, Mat(x), None, None, out, M, D))
    y = O.bf16_to_f32(out["y"].get())
    v = X.values(X.MXFP8, out["codes"].get(), out["scales"].get())
    assert np.all(np.abs(y[0] - 1) < 0.01)
    assert not y[1].any() and not v[1].any()
    tiny = wide(x[2:3]) / np.sqrt(EPS)
    assert np.all(np.abs(y[2] - tiny[0]) <= 2.0 ** -7 * tiny[0])
    assert np.all(np.abs(y[3] - 1) < 0.01) and np.all(np.abs(v[3] - 1) < 0.07)
    assert np.all(np.isnan(y[5])) and np.all(np.isnan(v[5]))
    # rstd of an infinite sum is 0: 0 elsewhere, inf * 0 at the infinity
    assert np.isnan(y[4, D - 1]) and not y[4, :D - 1].any()
    assert np.all(np.isnan(v[4, D - 32:])) and not v[4, :D - 32].any()


def test_eps_of_zero(ghip):
    x = bf(np.full((2, 64), 3.0))
    out = {"y": Mat.out(2, 64)}
    ok(ghip, call(ghip, Mat(x), None, None, out, 2, 64, 0.0))
    assert np.all(O.bf16_to_f32(out["y"].get()) == 1)


@pytest.mark.parametrize("M,D", [(1, 4096), (70, 1000), (520, 2048)])
def test_replayed_and_on_other_streams(ghip, M, D):
    """Norm and gradient captured into a graph, replayed with new inputs between eager calls on another stream."""
    rt = G.rt()
    st, other = rt.Stream(), rt.Stream()
    bufs = [G.empty(2 * M * D) for _ in range(5)] + [G.empty(2 * D) for _ in range(2)]
    x, r, y, s, dx, g, dg = bufs
    need = ghip.apus_ghip_rmsnorm_backward_ws(M, D)
    ws = [G.empty(need) for _ in range(2)]

    def both(stream, ws, dst):
        vp = G.vp
        ok(ghip, ghip.apus_ghip_rmsnorm_dev(vp(x), vp(r), vp(g), vp(dst[0]), vp(dst[1]), None, None, None, M, D, 0, 0, 0, 0, EPS, stream.vp))
        ok(ghip, ghip.apus_ghip_rmsnorm_backward_dev(vp(dst[0]), vp(g), None, vp(dst[1]), vp(r), vp(dst[2]), vp(dst[3]), M, D, 0, 0, 0, 0,
                                                     EPS, vp(ws), need, stream.vp))

    for b, v in zip((x, r, g), inputs(M, D, 6)):
        b.upload(v)
    mine, eager = (s, y, dx, dg), [G.empty(2 * M * D) for _ in range(3)] + [G.empty(2 * D)]
    graph = rt.Graph(st)
    graph.begin()
    both(st, ws[0], mine)
    graph.end()
    for k in range(4):
        for b, v in zip((x, r, g), inputs(M, D, 7, k)):
            b.upload(v)
        graph.launch()
        both(other, ws[1], eager)
        st.synchronize()
        other.synchronize()
        for a, b in zip(mine, eager):
            n = a.nbytes // 2
            assert np.array_equal(a.download(np.uint16, n), b.download(np.uint16, n))
    graph.close()


def test_the_same_bits_again(ghip):
    M, D = 1300, 2100
    s, ds, g, dy = inputs(M, D, 8)
    a, b = (run_grad(ghip, Mat(s), Mat(g), None, Mat(dy), Mat(ds), M, D) for _ in range(2))
    assert all(np.array_equal(a[k], b[k]) for k in a)


def test_many_rows(ghip):
    """More rows than one launch takes workgroups of a row."""
    M, D = (1 << 21) + 3, 1056
    x, y = G.empty(2 * M * D), G.empty(2 * M * D)
    ok(ghip, ghip.apus_synth_bf16_normal_dev(G.vp(x), M * D, 1, 2, 0, None))
    ok(ghip, ghip.apus_ghip_rmsnorm_dev(G.vp(x), None, None, None, G.vp(y), None, None, None, M, D, 0, 0, 0, 0, EPS, None))
    for row in (0, 1, (1 << 21) - 1, 1 << 21, M - 1):
        v = G.download_ptr(x.ptr + 2 * row * D, np.uint16, (1, D))
        want, err, _ = X.norm(wide(v), None, EPS)
        R.check(wide(G.download_ptr(y.ptr + 2 * row * D, np.uint16, (1, D))), want, err + X.HALF * np.abs(want), "row %d" % row)
