"""Products with MXFP4 weights where the other tests do not go: weight scales at both ends under BF16 x, microscaled x of
every size in the forms for few rows, the same bits from call to call, and every product and backward pass on two streams
at once."""
import numpy as np
import pytest

import ffn_ref as R
import gpu_util as G
import mx_ref as X
import oracle as O
from test_gpu_ffn import Mat, bf, ok, seed, wide
from test_gpu_mx import XTYPES, Act, Mx, acts, gated, linear, weights

pytestmark = pytest.mark.gpu

BYTES = np.array([0, 1, 2, 60, 127, 200, 253, 254])                 # a row's weight scales, 2^(byte - 127)


def ends(rng, N):
    """MXFP4 weights with these scales, all of them BF16 numbers: none past 2^128."""
    c = rng.integers(0, 8, (N, 256))
    c[:, 192:224] %= 6                                              # at most 3 * 2^126
    c[:, 224:] %= 4                                                 # at most 1.5 * 2^127
    c |= 8 * rng.integers(0, 2, (N, 256))
    return Mx(X.MXFP4, X.stored(X.MXFP4, c.astype(np.uint8)), np.tile(BYTES.astype(np.uint8), (N, 1)))


def against(rng, M):
    """BF16 x whose products with these weights are ordinary numbers."""
    e = np.maximum(127 - np.repeat(BYTES, 32), -125)
    return bf(np.ldexp(rng.choice([-1.0, 1.0], (M, 256)) * rng.uniform(0.5, 0.99, (M, 256)), e))


@pytest.mark.parametrize("M,N", [(1, 40), (2, 300), (16, 70), (130, 300)])
def test_bf16_x_past_weight_scales_at_both_ends(ghip, M, N):
    """Weights from 2^-128, below the normal BF16 numbers, up to 1.5 * 2^127, in the few rows' kernel and on tiles."""
    rng = seed(57, M, N)
    wg, wu, x = ends(rng, N), ends(rng, N), Act(X.BF16, against(rng, M))
    y, h = Mat.out(M, N), Mat.out(M, N)
    ok(ghip, linear(ghip, wg, x, None, None, y, R.NONE))
    R.check(wide(y.get()), *X.linear(x.values, wg.values, None, None, R.NONE, X.BF16), "linear")
    ok(ghip, gated(ghip, wg, wu, x, h, R.RELU, 0.0))
    R.check(wide(h.get()), *X.gated(x.values, wg.values, wu.values, R.RELU, 0.0, X.BF16), "gated")


@pytest.mark.parametrize("M", [2, 130])
def test_weights_that_bf16_does_not_hold(ghip, M):
    """Past 2^128 a weight is an infinity to BF16 x, in its own column only."""
    N = 40
    c = np.full((N, 64), 2, np.uint8)                               # 1
    c[7, 5] = 7                                                     # 6
    s = np.full((N, 4), 127, np.uint8)
    s[:, 2:] = 0
    s[7, 0] = 254
    w, x = Mx(X.MXFP4, X.stored(X.MXFP4, c), s), Act(X.BF16, bf(np.full((M, 64), 2.0 ** -100)))
    y, h = Mat.out(M, N), Mat.out(M, N)
    ok(ghip, linear(ghip, w, x, None, None, y, R.NONE))
    ok(ghip, gated(ghip, w, w, x, h, R.NONE, 0.0))
    for m in (y, h):
        got = O.bf16_to_f32(m.get())
        assert np.all(np.isposinf(got[:, 7])) and np.all(np.isfinite(np.delete(got, 7, 1)))


@pytest.mark.parametrize("xt", [X.MXFP8, X.MXFP4])
@pytest.mark.parametrize("M,N", [(2, 40), (16, 300)])
def test_scales_of_every_size_in_few_rows(ghip, M, N, xt):
    """Blocks of x from 2^-127 on against weights up to 2^120 in the gated kernel of few rows."""
    K = 256
    rng = seed(58, M, N, xt)
    cx = rng.integers(0, 256 if xt == X.MXFP8 else 16, (M, K)).astype(np.uint8)
    if xt == X.MXFP8:
        cx[cx & 0x7F == 0x7F] = 0
    e = np.array([0, 1, 7, 60, 127, 200, 246, 254])
    sx, sw = np.zeros((M, 8), np.uint8), np.zeros((N, 8), np.uint8)
    sx[:], sw[:] = e, np.minimum(254 - e, 246)
    wg, wu = (Mx(X.MXFP4, X.stored(X.MXFP4, rng.integers(0, 16, (N, K)).astype(np.uint8)), sw) for _ in range(2))
    x = Act.__new__(Act)
    x.mx = Mx(xt, X.stored(xt, cx), sx)
    x.type, x.args, x.ld, x.values = xt, (xt, G.vp(x.mx.codes), G.vp(x.mx.scales)), 0, x.mx.values
    h = Mat.out(M, N)
    ok(ghip, gated(ghip, wg, wu, x, h, R.RELU, 50.0))
    R.check(wide(h.get()), *X.gated(x.values, wg.values, wu.values, R.RELU, 50.0, xt), "gated")


def test_more_outputs_than_a_launch_takes(ghip):
    """Refused with a message; the addresses are not read."""
    P, most = 1 << 20, (1 << 31) - 1
    assert ghip.apus_ghip_mxfp4_linear_dev(P, P, 0, P, None, None, None, P, most, most, 32, 0, 0, 0, R.NONE, None) == 1
    said = ghip.apus_ghip_last_error().decode()
    assert "%d x %d" % (most, most) in said and "tiles" in said


def linear_backward(lib, w, x, bias, dy, out, ws, act, st=None):
    (M, N), K = (dy.rows, dy.cols), w.values.shape[1]
    ok(lib, lib.apus_ghip_mxfp4_linear_backward_dev(G.vp(w.codes), G.vp(w.scales), x.p, G.vp(bias), dy.p, out[0].p, out[1].p, M, N, K, x.ld, dy.ld,
                                                    out[0].ld, act, G.vp(ws), ws.nbytes, st))


def gated_backward(lib, wg, wu, x, dh, dx, ws, act, limit, st=None):
    (M, N), K = (dh.rows, dh.cols), wg.values.shape[1]
    ok(lib, lib.apus_ghip_mxfp4_gated_backward_dev(G.vp(wg.codes), G.vp(wg.scales), G.vp(wu.codes), G.vp(wu.scales), x.p, dh.p, dx.p, M, N, K, x.ld,
                                                   dh.ld, dx.ld, act, limit, G.vp(ws), ws.nbytes, st))


def products(lib, M, N, K):
    """(outputs(), run(outputs, stream)) of every product and backward pass of these sizes."""
    rng = seed(59, M, N, K)
    w, w2 = weights(rng, N, K), weights(rng, N, K)
    xs, dy = [Act(t, acts(rng, M, K)) for t in XTYPES], Mat(bf(rng.standard_normal((M, N))))
    bias, res = G.dev(bf(rng.standard_normal(N))), Mat(bf(rng.standard_normal((M, N))))
    sizes = lib.apus_ghip_mxfp4_linear_backward_ws(M, N, K), lib.apus_ghip_mxfp4_gated_backward_ws(M, N, K)

    def outputs():
        return {"y": [Mat.out(M, N) for _ in xs], "h": [Mat.out(M, N) for _ in xs], "dx": Mat.out(M, K), "db": Mat.out(1, N), "gx": Mat.out(M, K),
                "ws": [G.empty(n) for n in sizes]}

    def run(o, st=None):
        for x, y, h in zip(xs, o["y"], o["h"]):
            ok(lib, linear(lib, w, x, bias, res, y, R.GELU, st))
            ok(lib, gated(lib, w, w2, x, h, R.SILU, 1.5, st))
        linear_backward(lib, w, xs[0].mat, bias, dy, (o["dx"], o["db"]), o["ws"][0], R.SILU, st)
        gated_backward(lib, w, w2, xs[0].mat, dy, o["gx"], o["ws"][1], R.SILU, 1.5, st)

    return outputs, run


def results(o):
    return [m.get() for m in o["y"] + o["h"] + [o["dx"], o["db"], o["gx"]]]


@pytest.mark.parametrize("M,N,K", [(1, 4096, 1024), (5, 1040, 4096), (16, 300, 640), (300, 520, 640), (1024, 1032, 256)])
def test_called_again(ghip, M, N, K):
    """The same bits from call to call, of few rows and of many."""
    outputs, run = products(ghip, M, N, K)
    first = None
    for _ in range(4):
        o = outputs()
        run(o)
        got = results(o)
        assert first is None or all(np.array_equal(a, b) for a, b in zip(first, got))
        first = got


@pytest.mark.parametrize("M", [3, 300])
def test_all_products_on_two_streams_at_once(ghip, M):
    """Each with its own outputs and workspaces, against the same calls alone."""
    outputs, run = products(ghip, M, 520, 640)
    alone = outputs()
    run(alone)
    want, sts = results(alone), [G.rt().Stream() for _ in range(2)]
    outs = [outputs() for _ in sts]
    for _ in range(3):
        for st, o in zip(sts, outs):
            run(o, st.vp)
    for st, o in zip(sts, outs):
        st.synchronize()
        assert all(np.array_equal(a, b) for a, b in zip(want, results(o)))


@pytest.mark.parametrize("M", [3, 300])
def test_backward_passes_replayed(ghip, M):
    """Captured once, replayed between eager calls on another stream."""
    rt = G.rt()
    outputs, run = products(ghip, M, 264, 352)
    a, b, st, other = outputs(), outputs(), rt.Stream(), rt.Stream()
    run(b, other.vp)
    other.synchronize()
    want = results(b)
    graph = rt.Graph(st)
    graph.begin()
    run(a, st.vp)
    graph.end()
    for _ in range(4):
        graph.launch()
        run(b, other.vp)
        st.synchronize()
        other.synchronize()
        assert all(np.array_equal(x, y) for x, y in zip(want, results(a))) and all(np.array_equal(x, y) for x, y in zip(want, results(b)))
    graph.close()
