"""Every tile and every row form of the dense feed-forward products, run by
itself at shapes with ragged edges on all sides, against the 64-bit forms."""
import ctypes

import numpy as np
import pytest

import ffn_forms as F
import ffn_ref as R
import gpu_util as G
import oracle as O
import test_gpu_ffn as T
from test_gpu_ffn import Mat, bf, fp8, seed, wide

pytestmark = pytest.mark.gpu

TILES = {"linear": 8, "linear fp8": 6, "linear fp8 exact": 6, "gated": 9, "gated fp8": 6, "gated fp8 exact": 6, "dlinear": 9,
         "dgated": 8, "dx": 6, "dw": 4}


def addr(buf):
    return G.vp(buf).value


class Case:
    """Operands, outputs and the 64-bit result of one forward-shaped product."""

    def __init__(self, family, M, N, K, act, limit, pad=8):
        mode, self.w8, _, _ = F.FAMILIES[family]
        rng = seed(M, N, K, list(F.FAMILIES).index(family))
        x = bf(rng.standard_normal((M, K)))
        dual = mode in (F.GATED, F.DGATED)
        ws = []
        for _ in range(2 if dual else 1):
            if self.w8:
                codes, scales = fp8(rng, N, K, nans=self.w8 == 2)
                ws.append((G.dev(codes), G.dev(scales), wide(O.dequant(codes, scales))))
            else:
                w = bf(rng.standard_normal((N, K)) / np.sqrt(K))
                ws.append((G.dev(w), None, wide(w)))
        bias = bf(rng.standard_normal(N)) if not dual else None
        other = bf(rng.standard_normal((M, N))) if mode != F.GATED else None
        self.keep = ws, Mat(x, pad), None if bias is None else G.dev(bias), None if other is None else Mat(other, 3, 1)
        (_, xm, bd, om) = self.keep
        grad = mode in (F.DLINEAR, F.DGATED)
        self.cols = N
        wide_n = -(-N // 8) * 8 if grad else N                       # the gradients' own columns
        self.out = Mat.out(M, wide_n, 0 if grad else 5, 0 if grad else 1)
        self.out2 = Mat.out(M, wide_n) if mode == F.DGATED else None
        self.p = F.prod(family, M, N, K, a=xm.p.value, b=addr(ws[0][0]), b2=addr(ws[1][0]) if dual else None,
                        s=addr(ws[0][1]) if self.w8 else None, s2=addr(ws[1][1]) if self.w8 and dual else None, lda=xm.ld, ldb=K)
        self.ep = F.Ep(bias=None if bd is None else addr(bd), in_=None if om is None else om.p.value, out=self.out.p.value,
                       out2=None if self.out2 is None else self.out2.p.value, ldin=0 if om is None else om.ld, ldout=self.out.ld,
                       act=act, limit=limit or np.inf, pad=int(grad))
        xf, wf = wide(x), [w[2] for w in ws]
        bf64, of64 = None if bias is None else wide(bias), None if other is None else wide(other)
        if mode == F.LINEAR:
            self.want = [R.linear(xf, wf[0], bf64, of64, act)]
        elif mode == F.GATED:
            self.want = [R.gated(xf, wf[0], wf[1], act, limit)]
        elif mode == F.DLINEAR:
            self.want = R.dz_linear(xf, wf[0], bf64, of64, act)
        else:
            self.want = R.dz_gated(xf, wf[0], wf[1], of64, act, limit)

    def check(self, what):
        for m, (want, tol) in zip((self.out, self.out2), self.want):
            got = wide(m.get())
            assert not got[:, self.cols:].any(), what
            R.check(got[:, :self.cols], want, tol + 1e-38, what)


def forward(family, i):
    return R.ACTS[i % 5], (0.0, 1.5)[i % 2]


@pytest.mark.parametrize("family,tile", [(f, i) for f in F.ROWS for i in range(TILES[f])])
def test_tile(ghip, family, tile):
    assert len(F.tiles(ghip, family)) == TILES[family]
    t = F.tiles(ghip, family)[tile]
    mode, w8, _, _ = F.FAMILIES[family]
    for M, N, K in [(t.bm + 19, t.bn + 13, 400), (t.bm, 2 * t.bn, 64), (3, 8, 16), (2 * t.bm - 1, t.bn + 8, 1040),
                    (t.bm + 5, t.bn + 33, 72), (5, 40, 24), (t.bm, 2 * t.bn, 1096), (33, 130, 56), (70, 129, 168)]:
        c = Case(family, M, N, K, *forward(family, tile + M), pad=16 if w8 else 8)
        assert F.gemm_fits(ghip, family, c.p)
        assert ghip.ghip_launch_ffn_gemm(mode, tile, ctypes.c_uint32(1), ctypes.byref(c.p), ctypes.byref(c.ep), None) == 0
        c.check((family, tile, M, N, K))


@pytest.mark.parametrize("family,form", [(f, i) for f in F.ROWS for i in range(F.ROW_FORMS[f])])
def test_row_form(ghip, family, form):
    mode = F.FAMILIES[family][0]
    for M, N, K in [(1, 37, 24), (4, 131, 1032), (7, 64, 512), (16, 205, 2056), (65, 136, 328)]:
        c = Case(family, M, N, K, *forward(family, form + M))
        assert F.rows_fits(ghip, family, c.p)
        assert ghip.ghip_launch_ffn_rows(mode, form, ctypes.byref(c.p), ctypes.byref(c.ep), None) == 0
        c.check((family, form, M, N, K))


def sums(pairs):
    z = sum(a @ b.T for a, b in pairs)
    k = sum(a.shape[1] for a, _ in pairs)
    e = (k + 8) * 2.0 ** -24 * sum(np.abs(a) @ np.abs(b).T for a, b in pairs)
    return z, e + R.HALF * np.abs(z) + 1e-38


def laid(codes, slow):
    """A k-fast [rows, k] matrix as the family's operand lies in memory: rows of
    whole vectors, the pad zeros."""
    m = np.ascontiguousarray(codes.T if slow else codes)
    out = np.zeros((m.shape[0], -(-m.shape[1] // 8) * 8), np.uint16)
    out[:, :m.shape[1]] = m
    return G.dev(out), out.shape[1]


SPLITS = [1, 2, 3, 7]
TWO = [("dx", ""), ("dx", "pair"), ("dw", ""), ("dw", "batch")]  # dg Wg + du Wu; dWg and dWu


@pytest.mark.parametrize("splits", SPLITS)
@pytest.mark.parametrize("family,two,tile", [(f, w, i) for f, w in TWO for i in range(TILES[f])])
def test_gradient_tile(ghip, family, two, tile, splits):
    assert len(F.tiles(ghip, family)) == TILES[family]
    t, (_, _, slow_a, slow_b) = F.tiles(ghip, family)[tile], F.FAMILIES[family]
    for M, N, K in [(t.bm + 19, t.bn + 16, 395), (t.bm, 2 * t.bn, 512), (5, 8, 449)]:
        rng = seed(M, N, K, tile, splits)
        ab = [(bf(rng.standard_normal((M, K))), bf(rng.standard_normal((N, K)) / np.sqrt(K))) for _ in range(2 if two else 1)]
        if two == "batch":
            ab[1] = ab[1][0], ab[0][1]                              # dz_g and dz_u of one x
        dev = [(laid(a, slow_a), laid(b, slow_b)) for a, b in ab]
        (da, lda), (db, ldb) = dev[0]
        more = {} if not two else dict(a2=addr(dev[1][0][0]), b2=addr(dev[1][1][0]))
        size = splits * M * (-(-N // 8) * 8) * 4 * (2 if two == "batch" else 1)
        part = G.dev(np.full(size // 4 + 64, np.nan, np.float32))
        p = F.prod(family, M, N, K, a=addr(da), b=addr(db), lda=lda, ldb=ldb, apad=1, batch=int(two == "batch"), part=addr(part),
                   part_bytes=size, **more)
        outs = [Mat.out(M, N, 3, 1) for _ in range(2 if two == "batch" else 1)]
        e = F.Ep(out=outs[0].p.value, out2=outs[-1].p.value, ldout=outs[0].ld)
        assert F.gemm_fits(ghip, family, p)
        assert ghip.ghip_launch_ffn_gemm(F.STORE, tile, ctypes.c_uint32(splits), ctypes.byref(p), ctypes.byref(e), None) == 0
        pairs = [ab] if two == "pair" else [[x] for x in ab]
        for out, of in zip(outs, pairs):
            want, tol = sums([(wide(a), wide(b)) for a, b in of])
            R.check(wide(out.get()), want, tol, (family, tile, M, N, K, splits, two))
        assert np.isnan(G.host(part, np.float32, size // 4 + 64)[size // 4:]).all()


@pytest.mark.parametrize("pair", range(F.PAIRS))
@pytest.mark.parametrize("sx,sw", [(1, 1), (3, 1), (1, 2)])
@pytest.mark.parametrize("two", [0, 1])
@pytest.mark.parametrize("M,N,K", [(200, 264, 192), (395, 129, 328), (130, 8, 1032)])
def test_pair(ghip, pair, sx, sw, two, M, N, K):
    """dx, dW and dbias in one launch: any of them in pieces of k."""
    pr = F.pairs(ghip)[pair]
    tiles = [[t for t in F.tiles(ghip, f) if (t.bm, t.bn, t.lds) == tuple(w)][0] for f, w in (("dx", pr.dx), ("dw", pr.dw))]
    rng = seed(M, N, K, two, pair)
    dz, w = [bf(rng.standard_normal((M, N))) for _ in range(1 + two)], [bf(rng.standard_normal((N, K)) / np.sqrt(K)) for _ in range(1 + two)]
    x = bf(rng.standard_normal((M, K)))
    dzd, wd, xd = [laid(z, 0) for z in dz], [G.dev(v) for v in w], G.dev(x)
    ld = dzd[0][1]
    stages = -(-N // 64) * (1 + two), -(-M // 64)
    sx, sw = min(sx, stages[0]), min(sw, stages[1])
    cells = sx * M * K if sx > 1 else sw * N * K * (1 + two)
    part = G.dev(np.full(cells + 64, np.nan, np.float32))
    more = lambda a, b: dict(a2=addr(a[0]), b2=addr(b)) if two else {}  # noqa: E731
    px = F.prod("dx", M, K, N, a=addr(dzd[0][0]), b=addr(wd[0]), lda=ld, apad=1, splits=sx, part=addr(part) if sx > 1 else None,
                **more(dzd[-1], wd[-1]))
    pw = F.prod("dw", N, K, M, a=addr(dzd[0][0]), b=addr(xd), lda=ld, apad=1, batch=two, splits=sw, part=addr(part) if sw > 1 else None,
                **more(dzd[-1], xd))
    dx, dw, db = Mat.out(M, K, 3, 1), [Mat.out(N, K) for _ in range(1 + two)], Mat.out(1, N)
    ex, ew = F.Ep(out=dx.p.value, ldout=dx.ld), F.Ep(out=dw[0].p.value, out2=dw[-1].p.value, ldout=K)
    sm = F.Sum(dz=addr(dzd[0][0]), ld=ld, M=M, N=N, out=db.p.value)
    at = lambda s: ctypes.cast(ctypes.byref(s), ctypes.c_void_p)    # noqa: E731
    pr.launch(at(px), at(ex), at(pw), at(ew), at(sm), at(tiles[0]), at(tiles[1]), None)
    f = G.host(part, np.float32, cells + 64)
    assert np.isnan(f[cells:]).all()
    grads = R._grads(wide(x), [(wide(v), wide(z), np.zeros((M, N))) for v, z in zip(w, dz)])
    if sx > 1:                                                      # the sums that would be joined
        got = f[:cells].reshape(sx, M, K).astype(np.float64).sum(0)
        assert np.all(np.abs(got - grads["dx"][0]) <= grads["dx"][1]) and (dx.get() == 0x7E57).all()
    else:
        R.check(wide(dx.get()), *grads["dx"], "dx")
    for i, m in enumerate(dw):
        if sw > 1:
            got = f[:cells].reshape(1 + two, sw, N, K)[i].astype(np.float64).sum(0)
            assert np.all(np.abs(got - grads["dw%d" % i][0]) <= grads["dw%d" % i][1]) and (m.get() == 0x7E57).all()
        else:
            R.check(wide(m.get()), *grads["dw%d" % i], "dw%d" % i)
    R.check(wide(db.get())[0], *grads["db"], "db")


# M, N, K, two: a pair alone, with dx split, with dW split, with the sum in a launch of its own; two launches; rows of odd widths
BACKWARDS = [(300, 512, 256, 0), (57, 3400, 1472, 1), (2165, 72, 288, 1), (1200, 96, 264, 0), (600, 2048, 2048, 1), (333, 129, 72, 0),
             (90, 257, 136, 1)]


@pytest.mark.parametrize("M,N,K,two", BACKWARDS)
def test_gradients_of_the_entries(ghip, M, N, K, two):
    rng = seed(M, N, K, two, 77)
    x, w = bf(rng.standard_normal((M, K))), [bf(rng.standard_normal((N, K)) / np.sqrt(K)) for _ in range(1 + two)]
    dy = bf(rng.standard_normal((M, N)))
    if two:
        got = T.run_gated_bwd(ghip, G.dev(w[0]), G.dev(w[1]), Mat(x), Mat(dy), M, N, K, R.SILU, 0.0)
        want = R.gated_backward(wide(x), wide(w[0]), wide(w[1]), wide(dy), R.SILU, 0.0)
        names = {"dx": "dx", "dwg": "dw0", "dwu": "dw1"}
    else:
        got = T.run_linear_bwd(ghip, G.dev(w[0]), Mat(x), None, Mat(dy), M, N, K, R.GELU)
        want = R.linear_backward(wide(x), wide(w[0]), None, wide(dy), R.GELU)
        names = {"dx": "dx", "dw": "dw0", "db": "db"}
    for a, b in names.items():
        v, tol = want[b]
        R.check(wide(got[a]).reshape(v.shape), v, tol, (M, N, K, a))
