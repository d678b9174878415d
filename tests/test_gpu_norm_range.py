"""The norm and its gradient over rows of every size that BF16 holds: squares and products that are no f32 numbers by
themselves, with an eps of 0 or one as small as the rows."""
import numpy as np
import pytest

import ffn_ref as R
import gpu_util as G
import mx_ref as X
import oracle as O
from test_gpu_ffn import Mat, bf, ok, seed, wide
from test_gpu_norm import Bytes, call, check_mx, f32s, get_f32, inputs, run_grad

pytestmark = pytest.mark.gpu

# one of each form: a wave or a workgroup a row, one piece a thread or several, a row read twice
COLUMNS = [96, 1000, 2048, 4096, 8000, 16000, 17024]


def scaled(x, e):
    """Row m of x times 2^e[m]."""
    return bf(np.ldexp(O.bf16_to_f32(x).astype(np.float64), np.asarray(e)[:, None]).astype(np.float32))


@pytest.mark.parametrize("D", COLUMNS)
@pytest.mark.parametrize("eps", [0.0, 2.0 ** -118])
def test_norm_of_rows_of_any_size(ghip, D, eps):
    """From rows near the least normal number to rows near the largest one, and a row of the least number of all; an eps of
    2^-118 counts for rows of 2^-59."""
    e = [-120, -101, -76, -64, -59, -52, -49, 0, 49, 61, 64, 90, 118]
    M = len(e) + 1
    x, _, g, _ = inputs(M, D, 11)
    x = scaled(x, e + [0])
    x[M - 1] = 1                                                    # 2^-133
    out = {"y": Mat.out(M, D), "rstd": f32s(M)}
    if D % 32 == 0:
        out |= {"codes": Bytes(M, D), "scales": Bytes(M, X.scale_ld(D))}
    ok(ghip, call(ghip, Mat(x), None, Mat(g), out, M, D, eps))
    y, err, rstd = X.norm(wide(x), wide(g)[0], eps)
    R.check(wide(out["y"].get()), y, err + X.HALF * np.abs(y), "y")
    got = get_f32(out["rstd"])
    assert np.all(np.abs(got[:-1] - rstd[:-1]) <= ((D + 8) / 2 + 6) * X.U * rstd[:-1])
    if eps == 0.0:
        assert np.isinf(got[-1])                                    # 2^133 is no f32
    if D % 32 == 0:
        check_mx(out["codes"].get(), out["scales"].get(), y, err)


@pytest.mark.parametrize("D", [96, 4096, 17024])
def test_rows_of_zeros_with_an_eps_of_zero(ghip, D):
    """0 / 0, in its own row only."""
    x = bf(np.ones((3, D)))
    x[1] = 0
    out = {"y": Mat.out(3, D)}
    ok(ghip, call(ghip, Mat(x), None, None, out, 3, D, 0.0))
    y = O.bf16_to_f32(out["y"].get())
    assert np.all(np.isnan(y[1])) and np.all(y[[0, 2]] == 1)


@pytest.mark.parametrize("M,D", [(13, D) for D in COLUMNS] + [(1030, D) for D in COLUMNS[:4]])
@pytest.mark.parametrize("given", [False, True])
def test_gradient_of_rows_of_any_size(ghip, M, D, given):
    """dy of a size between its row's and 1, so that their products leave the f32 range and dx does not; few rows and more than
    one launch's form takes."""
    s, ds, g, dy = inputs(M, D, 12)
    e = np.resize([-110, -90, -64, -50, 0, 45, 64, 88, 110], M)
    s, dy, ds = scaled(s, e), scaled(dy, e // 2), scaled(ds, e // 2 - e)
    rstd = G.dev((1 / np.sqrt((wide(s) ** 2).mean(1))).astype(np.float32)) if given else None
    got = run_grad(ghip, Mat(s), Mat(g), rstd, Mat(dy), Mat(ds), M, D, eps=0.0)
    dx, dg = X.norm_backward(wide(s), wide(g)[0], wide(dy), wide(ds), 0.0)
    R.check(wide(got["dx"]), *dx, "dx")
    R.check(wide(got["dgamma"])[0], *dg, "dgamma")


def test_gradient_by_differences(ghip):
    """dx of tiny and huge rows against differences of the norm's 64-bit form."""
    M, D = 4, 64
    rng = seed(56)
    s, dy = scaled(bf(rng.standard_normal((M, D))), [-100, -70, 70, 100]), bf(rng.standard_normal((M, D)))
    dy = scaled(dy, [-50, -35, 35, 50])
    got = wide(run_grad(ghip, Mat(s), None, None, Mat(dy), None, M, D, eps=0.0)["dx"])
    v, d = wide(s), wide(dy)
    step = np.sqrt((v * v).mean(1, keepdims=True)) * 1e-4
    for c in range(0, D, 7):
        h = np.zeros((M, D))
        h[:, c:c + 1] = step
        want = ((X.norm(v + h, None, 0.0)[0] - X.norm(v - h, None, 0.0)[0]) * d).sum(1) / (2 * step[:, 0])
        # the differences' own error is of the step's square, 1e-8 of the terms; dx is rounded once
        size = np.abs(d).sum(1) / np.sqrt((v * v).mean(1))
        assert np.all(np.abs(got[:, c] - want) <= X.HALF * np.abs(want) + 1e-5 * size)
