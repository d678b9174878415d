"""Which kernel a product with MXFP4 weights takes: the picks need no device."""
import ctypes
import math
import random

import pytest

import mx_forms as F

AT = 1 << 20                                                        # never read


def picks(lib, mode, xt, M, N, K):
    """((tile, us), (form, us)); -1: none."""
    p, out = F.prod(xt, M, N, K, AT, AT, AT, AT, AT if mode == F.GATED else None, AT if mode == F.GATED else None), []
    for f in (lib.ghip_mx_gemm_pick, lib.ghip_mx_rows_pick):
        us = ctypes.c_float()
        out.append((f(mode, ctypes.byref(p), ctypes.byref(us)), us.value))
    return out


def pick(lib, mode, xt, M, N, K):
    (tile, a), (form, b) = picks(lib, mode, xt, M, N, K)
    return ("rows", form) if form >= 0 and (tile < 0 or b <= a) else ("tiles", tile)


@pytest.fixture(scope="module")
def lib(pkg):
    return pkg.load()


@pytest.mark.parametrize("mode", [F.LINEAR, F.GATED])
@pytest.mark.parametrize("xt", [0, 1, 2])
def test_every_kernel_is_the_pick_of_some_shape(lib, mode, xt):
    rng, got = random.Random(3), set()
    draw = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))  # noqa: E731
    for _ in range(6000):
        got.add(pick(lib, mode, xt, draw(1, 16384), draw(16, 16384), 32 * draw(1, 512)))
    # a family's tiles serve both modes: each is the pick of one of them
    other = F.GATED if mode == F.LINEAR else F.LINEAR
    for _ in range(6000):
        kind, form = pick(lib, other, xt, draw(1, 16384), draw(16, 16384), 32 * draw(1, 512))
        if kind == "tiles":
            got.add((kind, form))
    assert got == {("rows", i) for i in range(F.rows(lib, mode, xt))} | {("tiles", i) for i in range(F.tiles(lib, mode, xt))}


@pytest.mark.parametrize("mode", [F.LINEAR, F.GATED])
@pytest.mark.parametrize("xt", [0, 1, 2])
def test_few_rows_stream_and_many_take_tiles(lib, mode, xt):
    for N, K in [(4096, 4096), (12288, 4096), (4096, 12288)]:
        # the linear has no row forms
        few = "tiles" if mode == F.LINEAR else "rows"
        assert all(pick(lib, mode, xt, M, N, K)[0] == few for M in (1, 4, 16))
        assert pick(lib, mode, xt, 4096, N, K)[0] == "tiles"


@pytest.mark.parametrize("xt", [0, 1, 2])
def test_what_each_kind_takes(lib, xt):
    """A k too long for a row of x in LDS goes to tiles, one too long for their offsets to rows or nowhere; outputs of more
    workgroups than a launch takes go to rows."""
    assert picks(lib, F.GATED, xt, 1, 64, 1 << 21)[1][0] == -1 and pick(lib, F.GATED, xt, 1, 64, 1 << 21)[0] == "tiles"
    assert pick(lib, F.GATED, xt, 1, 64, 1 << 24) == ("tiles", -1)
    assert picks(lib, F.GATED, xt, (1 << 31) - 1, (1 << 31) - 1, 32)[0][0] == -1
    assert pick(lib, F.GATED, xt, (1 << 31) - 1, (1 << 31) - 1, 32)[0] == "rows"
    # what the entries let through has a kernel: any stride up to k of 2^15 (not the linear's with BF16 x), less than 2^22
    # elements to 2^22
    for mode in (F.LINEAR, F.GATED):
        far = (1 << 22) - 8 if (mode, xt) == (F.LINEAR, 0) else 1 << 30
        for M, K, ld in [(1, 1 << 15, far), (4096, 1 << 15, far), (1, (1 << 22) - 32, (1 << 22) - 32), (4096, (1 << 22) - 32, (1 << 22) - 8)]:
            p = F.prod(xt, M, 64, K, AT, AT, AT, AT, AT, AT)
            p.xld = 2 * ld if xt == 0 else K if xt == 1 else K // 2
            us = ctypes.c_float()
            assert max(f(mode, ctypes.byref(p), ctypes.byref(us)) for f in (lib.ghip_mx_gemm_pick, lib.ghip_mx_rows_pick)) >= 0
    assert all(us > 2.0 for _, us in picks(lib, F.GATED, xt, 1, 1, 32))
