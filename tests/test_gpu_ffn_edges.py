"""Calls of the dense feed-forward entries that the documentation allows at the
ends of their range: very many outputs, rows and products, the per-thread
stream, the same matrix twice, split and paired backward passes on two streams
and in graphs, dy of any alignment without an activation."""
import ctypes

import numpy as np
import pytest

import ffn_ref as R
import gpu_util as G
from test_gpu_ffn import Mat, bf, call_gated, call_linear, data, dev_w, ok, run_gated_bwd, run_linear_bwd, seed, wide

pytestmark = pytest.mark.gpu


def rows_of(buf, width, rows):
    return np.stack([G.download_ptr(G.vp(buf).value + 2 * m * width, np.uint16, (width,)) for m in rows])


@pytest.mark.parametrize("weights", ["bf16", "fp8"])
def test_more_than_2_31_outputs(ghip, weights):
    M, N, K = 65544, 32776, 16
    free, _ = G.rt().mem_info()
    if free < 3 * M * N * 2:
        pytest.skip("needs %d GiB of device memory" % (3 * M * N * 2 >> 30))
    x, [w, w2] = data(M, N, K, weights, "gated", seed(40))
    xd, wd, w2d, y = Mat(x), dev_w(w), dev_w(w2), G.empty(M * N * 2)
    out = type("Out", (), {"p": G.vp(y), "ld": N})
    at = [0, 255, 256, 32767, 65535, 65536, M - 1]
    ok(ghip, call_linear(ghip, wd, xd, None, None, out, M, N, K, R.RELU))
    R.check(wide(rows_of(y, N, at)), *R.linear(wide(x[at]), w[2], None, None, R.RELU), "linear")
    ok(ghip, call_gated(ghip, wd, w2d, xd, out, M, N, K, R.SILU, 1.0))
    R.check(wide(rows_of(y, N, at)), *R.gated(wide(x[at]), w[2], w2[2], R.SILU, 1.0), "gated")
    y.close()


@pytest.mark.parametrize("weights", ["bf16", "fp8"])
@pytest.mark.parametrize("M", [3, 70])
def test_a_long_k(ghip, M, weights):
    N, K = 24, (1 << 20) + 16
    x, [w] = data(M, N, K, weights, "linear", seed(41, M))
    y = Mat.out(M, N)
    ok(ghip, call_linear(ghip, dev_w(w), Mat(x), None, None, y, M, N, K, R.NONE))
    R.check(wide(y.get()), *R.linear(wide(x), w[2], None, None, R.NONE), "linear")


def test_many_rows(ghip):
    M, N, K = 200003, 8, 16
    rng = seed(42)
    x, [w, w2] = data(M, N, K, "bf16", "gated", rng)
    xd, dy, a, b = Mat(x), Mat(bf(rng.standard_normal((M, N)))), dev_w(w), dev_w(w2)
    y, h = Mat.out(M, N), Mat.out(M, N)
    ok(ghip, call_linear(ghip, a, xd, None, None, y, M, N, K, R.SILU))
    R.check(wide(y.get()), *R.linear(wide(x), w[2], None, None, R.SILU), "linear")
    ok(ghip, call_gated(ghip, a, b, xd, h, M, N, K, R.SILU, 0.0))
    R.check(wide(h.get()), *R.gated(wide(x), w[2], w2[2], R.SILU, 0.0), "gated")
    got = run_linear_bwd(ghip, a[0], xd, None, dy, M, N, K, R.SILU)
    want = R.linear_backward(wide(x), w[2], None, wide(dy.get()), R.SILU)
    for k, v in (("dx", "dx"), ("dw", "dw0")):
        R.check(wide(got[k]), *want[v], k)
    R.check(wide(got["db"])[0], *want["db"], "db")


def test_the_per_thread_stream(ghip):
    M, N, K = 40, 264, 128
    x, [w] = data(M, N, K, "bf16", "linear", seed(43))
    xd, wd, y = Mat(x), dev_w(w), Mat.out(M, N)
    G.rt().synchronize()
    ok(ghip, call_linear(ghip, wd, xd, None, None, y, M, N, K, R.GELU, st=ctypes.c_void_p(2)))
    G.rt().synchronize()
    R.check(wide(y.get()), *R.linear(wide(x), w[2], None, None, R.GELU), "linear")


@pytest.mark.parametrize("M,N,K", [(5, 264, 256), (90, 392, 320)])
def test_one_matrix_as_both_projections(ghip, M, N, K):
    rng = seed(44, M)
    x, [w] = data(M, N, K, "bf16", "linear", rng)
    dh, xd, wd, h = bf(rng.standard_normal((M, N))), Mat(x), dev_w(w), Mat.out(M, N)
    ok(ghip, call_gated(ghip, wd, wd, xd, h, M, N, K, R.GELU, 0.0))
    R.check(wide(h.get()), *R.gated(wide(x), w[2], w[2], R.GELU, 0.0), "gated")
    got = run_gated_bwd(ghip, wd[0], wd[0], xd, Mat(dh), M, N, K, R.GELU, 0.0)
    want = R.gated_backward(wide(x), w[2], w[2], wide(dh), R.GELU, 0.0)
    for k, v in (("dx", "dx"), ("dwg", "dw0"), ("dwu", "dw1")):
        R.check(wide(got[k]), *want[v], k)


# dx and dW in a launch, with dx split, dW split, dbias behind it, and apart
PASSES = [(2, 57, 3400, 1472), (2, 2165, 72, 288), (1, 1200, 96, 264), (1, 300, 512, 256), (2, 600, 2048, 1024)]


@pytest.mark.parametrize("two,M,N,K", PASSES)
def test_two_backward_passes_at_once(ghip, two, M, N, K):
    """Each on a stream and in a workspace of its own, eagerly and as graphs
    replayed with eager work between: the bits of a call alone."""
    rt, cases = G.rt(), []
    for k in range(2):
        rng = seed(45, M, k)
        x, ws = data(M, N, K, "bf16", "gated" if two == 2 else "linear", rng)
        xd, dy, wd = Mat(x), Mat(bf(rng.standard_normal((M, N)))), [G.dev(w[0]) for w in ws]
        if two == 2:
            got = run_gated_bwd(ghip, wd[0], wd[1], xd, dy, M, N, K, R.SILU, 2.0)
            names, need = ("dx", "dwg", "dwu"), ghip.apus_ghip_gated_backward_ws(M, N, K)
            out = [Mat.out(M, K), Mat.out(N, K), Mat.out(N, K)]
        else:
            got = run_linear_bwd(ghip, wd[0], xd, None, dy, M, N, K, R.SILU)
            names, need = ("dx", "dw", "db"), ghip.apus_ghip_linear_ep_backward_ws(M, N, K)
            out = [Mat.out(M, K), Mat.out(N, K), Mat.out(1, N)]
        work, st = Mat.out(1, need // 2), rt.Stream()

        def call(wd=wd, xd=xd, dy=dy, out=out, work=work, st=st, need=need):
            o = [m.p for m in out]
            if two == 2:
                ok(ghip, ghip.apus_ghip_bf16_gated_backward_dev(G.vp(wd[0]), G.vp(wd[1]), xd.p, dy.p, *o, M, N, K, 0, 0, 0, R.SILU, 2.0,
                                                                 work.p, need, st.vp))
            else:
                ok(ghip, ghip.apus_ghip_bf16_linear_ep_backward_dev(G.vp(wd[0]), xd.p, None, dy.p, *o, M, N, K, 0, 0, 0, R.SILU, work.p,
                                                                     need, st.vp))
        cases.append((call, out, [got[n] for n in names], st, work))

    def check():
        for _, _, _, st, _ in cases:
            st.synchronize()
        for _, out, want, _, work in cases:
            assert all(np.array_equal(o.get(), v) for o, v in zip(out, want))
            work.get()
            for o in out:
                o.buf.upload(o.before)
        rt.synchronize()
    for _ in range(3):
        for call, *_ in cases:
            call()
    check()
    graphs = []
    for call, _, _, st, _ in cases:
        gr = rt.Graph(st)
        gr.begin()
        call()
        gr.end()
        graphs.append(gr)
    for _ in range(3):
        for gr in graphs:
            gr.launch()
        check()
        cases[0][0]()                                               # eager work between the replays
        cases[0][3].synchronize()
    for gr in graphs:
        gr.close()


@pytest.mark.parametrize("M,N,K", [(300, 515, 200), (40, 264, 136), (700, 96, 72)])
@pytest.mark.parametrize("pad,off", [(0, 0), (8, 8), (3, 1), (5, 0)])
@pytest.mark.parametrize("room", [False, True])
def test_no_activation_backward_of_any_dy(ghip, M, N, K, pad, off, room):
    """dz is dy itself: with a workspace (laid out again where it is misaligned)
    and without."""
    rng = seed(46, M, pad)
    x, [w] = data(M, N, K, "bf16", "linear", rng)
    dy = bf(rng.standard_normal((M, N)))
    dyd, xd, wd = Mat(dy, pad, off), Mat(x), G.dev(w[0])
    out = [Mat.out(M, K, 3, 1), Mat.out(N, K), Mat.out(1, N)]
    need = ghip.apus_ghip_linear_ep_backward_ws(M, N, K)
    ws = Mat.out(1, need // 2)
    ok(ghip, ghip.apus_ghip_bf16_linear_ep_backward_dev(G.vp(wd), xd.p, None, dyd.p, *[o.p for o in out], M, N, K, 0, dyd.ld, out[0].ld,
                                                         R.NONE, ws.p if room else None, need if room else 0, None))
    want = R.linear_backward(wide(x), w[2], None, wide(dy), R.NONE)
    R.check(wide(out[0].get()), *want["dx"], "dx")
    R.check(wide(out[1].get()), *want["dw0"], "dw")
    R.check(wide(out[2].get())[0], *want["db"], "db")
    ws.get()
    assert np.array_equal(dyd.get(), dy)
