"""Which kernel a dense feed-forward product takes (no device: the estimates and
conditions are host code), for 256 CUs."""
import ctypes
import math
import random

import pytest

import ffn_forms as F


@pytest.fixture(scope="module")
def lib(pkg):
    return pkg.load()


def shapes(n, seed, most=16384):
    rnd = random.Random(seed)

    def size(lo):
        return round(math.exp(rnd.uniform(math.log(lo), math.log(most))))
    for _ in range(n):
        yield size(1), max(16, size(64) // 16 * 16), max(16, size(64) // 16 * 16)


def product(lib, family, M, N, K):
    """The product that a block of M rows, N outputs and K inputs makes, with the
    workspace that the backward entries give it."""
    dims = (M, K, N) if family == "dx" else (N, K, M) if family == "dw" else (M, N, K)
    p = F.prod(family, *dims, apad=int(family in ("dx", "dw")))
    if family in ("dx", "dw"):
        p.part_bytes = F.part_bytes(lib, *dims)
        p.part = F.AT if p.part_bytes else None
    return p


@pytest.mark.parametrize("family", F.FAMILIES)
def test_every_form_is_some_shapes_choice(lib, family):
    taken = {F.route(lib, family, product(lib, family, *s))[:2] for s in shapes(12000, 5)}
    want = {("tile", i) for i in range(len(F.tiles(lib, family)))}
    if family in F.ROWS:
        want |= {("rows", i) for i in range(F.ROW_FORMS[family])}
    assert taken == want


@pytest.mark.parametrize("family", ["dx", "dw"])
def test_splits_keep_their_limits(lib, family):
    split = 0
    for s in shapes(4000, 6):
        p = product(lib, family, *s)
        _, splits, _ = F.gemm_pick(lib, family, p)
        stages = (p.K + 63) // 64
        assert 1 <= splits <= 16 and (splits == 1 or stages // splits >= 8)
        if splits > 1:
            split += 1
            assert splits * p.M * p.N * 4 <= p.part_bytes <= (32 << 20) + 255
    assert split > 100
    p = product(lib, family, 64, 8192, 64) if family == "dx" else product(lib, family, 8192, 64, 64)
    assert F.gemm_pick(lib, family, p)[1] > 1
    p.part, p.part_bytes = None, 0
    assert F.gemm_pick(lib, family, p)[1] == 1


def test_estimates_grow_with_the_work(lib):
    for family in F.FAMILIES:
        for M, N, K in [(1, 512, 512), (300, 2048, 1536), (4096, 4096, 4096)]:
            base = F.gemm_pick(lib, family, F.prod(family, M, N, K))[2]
            assert 3.0 < base < F.gemm_pick(lib, family, F.prod(family, M, N, 4 * K))[2]
            assert base < F.gemm_pick(lib, family, F.prod(family, 64 * M, 4 * N, K))[2]


def test_many_outputs_take_tiles(lib):
    """More than 2^31 outputs: the largest tiles' grids are launches, the small ones' are not."""
    for family in F.FAMILIES:
        for M, N in [(16384, 154880), (1 << 20, 1 << 14)]:
            p = F.prod(family, M, N, 256)
            assert F.route(lib, family, p)[0] == "tile", (family, M, N)
            t = F.tiles(lib, family)[F.gemm_pick(lib, family, p)[0]]
            assert -(-M // t.bm) * -(-N // t.bn) * 256 < 1 << 32
    p = F.prod("linear", 0x7fffffff, 0x7ffffff8, 64)
    assert F.gemm_pick(lib, "linear", p)[0] == -1


MISALIGNED = [dict(a=F.AT + 2), dict(b=F.AT + 8), dict(lda=1028), dict(ldb=1032 + 4), dict(K=1028), dict(lda=1 << 22)]


@pytest.mark.parametrize("args", MISALIGNED, ids=lambda a: "-".join(a))
def test_what_direct_loads_cannot_take(lib, args):
    """Offsets of 31 bits, whole 16-byte pieces; the rest goes to the general kernel."""
    for family in ("linear", "dlinear", "gated", "dgated"):
        ok = dict(M=256, N=512, K=1024)
        assert F.gemm_fits(lib, family, F.prod(family, **ok))
        assert not F.gemm_fits(lib, family, F.prod(family, **{**ok, **args}))
    for w8 in ("linear fp8", "gated fp8 exact"):
        assert F.gemm_fits(lib, w8, F.prod(w8, 256, 512, 1032)) and F.gemm_fits(lib, w8, F.prod(w8, 256, 512, 24))
        assert not F.gemm_fits(lib, w8, F.prod(w8, 256, 512, 1028))
        assert not F.gemm_fits(lib, w8, F.prod(w8, 256, 512, 8))    # a half piece alone
        assert not F.gemm_fits(lib, w8, F.prod(w8, 256, 512, 1032, b=F.AT + 8))


def test_what_rows_can_take(lib):
    for family in F.ROWS:
        assert F.rows_fits(lib, family, F.prod(family, 4, 100, 1032))
        assert F.rows_fits(lib, family, F.prod(family, 4, 100, 1024, lda=4096))
        for bad in (dict(K=1028), dict(lda=1028), dict(a=F.AT + 8), dict(b=F.AT + 8), dict(lda=(1 << 24) + 8)):
            assert not F.rows_fits(lib, family, F.prod(family, **{**dict(M=4, N=100, K=1024), **bad}))
    for family in ("linear fp8", "gated fp8"):                       # the half piece needs a whole one
        assert not F.rows_fits(lib, family, F.prod(family, 4, 100, 8)) and F.rows_fits(lib, family, F.prod(family, 4, 100, 24))
    for family in ("dx", "dw"):
        assert not F.rows_fits(lib, family, F.prod(family, 4, 96, 1024))


def test_dw_reads_rows_of_any_width_where_they_are_padded(lib):
    """dz of N columns in rows of whole vectors: dW's A operand."""
    assert F.gemm_fits(lib, "dw", F.prod("dw", 515, 256, 300, lda=520, apad=1))
    assert not F.gemm_fits(lib, "dw", F.prod("dw", 515, 256, 300, lda=520))
    assert not F.gemm_fits(lib, "dw", F.prod("dw", 515, 250, 300, lda=520, ldb=256, apad=1))
    assert F.gemm_fits(lib, "dx", F.prod("dx", 300, 256, 515, lda=520, apad=1))
    assert not F.gemm_fits(lib, "dx", F.prod("dx", 300, 256, 515, lda=520))


def test_launchers_refuse_before_the_device(lib):
    e = F.Ep(out=F.AT, ldout=512)
    p = F.prod("dx", 256, 512, 1024, part=F.AT, part_bytes=2 * 256 * 512 * 4)

    def gemm(tile, splits, p=p):
        return lib.ghip_launch_ffn_gemm(F.STORE, tile, ctypes.c_uint32(splits), ctypes.byref(p), ctypes.byref(e), None)
    assert gemm(-1, 1) and gemm(99, 1) and gemm(0, 0)
    assert gemm(0, 3)                                               # three sums in room for two
    p.part = F.AT + 8
    assert gemm(0, 2)
    p.part = None
    assert gemm(0, 2)
    q = F.prod("dx", 256, 512, 64, part=F.AT, part_bytes=1 << 30)
    assert gemm(0, 2, q)                                            # one stage
    r = F.prod("linear", 4, 512, 1024)
    for form in (-1, 99):
        assert lib.ghip_launch_ffn_rows(F.LINEAR, form, ctypes.byref(r), ctypes.byref(e), None)
    assert lib.ghip_launch_ffn_rows(F.STORE, 0, ctypes.byref(p), ctypes.byref(e), None)


def block(lib, M, N, K, two):
    """The dx and dW products of a backward pass, in one workspace."""
    n, ld = 2 if two else 1, -(-N // 8) * 8
    more = dict(a2=F.AT, b2=F.AT) if two else {}
    dx, dw = F.prod("dx", M, K, N, lda=ld, apad=1, **more), F.prod("dw", N, K, M, lda=ld, apad=1, batch=int(two), **more)
    room = max(F.part_bytes(lib, M, K, n * N), F.part_bytes(lib, n * N, K, M))
    for p in (dx, dw):
        p.part, p.part_bytes = F.AT if room else None, room
    return dx, dw


def test_pairs(lib):
    """Every pair is some backward pass's choice, alone and with either product
    split, never with both; its tiles are in the tables."""
    pairs = F.pairs(lib)
    assert len(pairs) == F.PAIRS
    taken, apart = set(), 0
    for i, (M, N, K) in enumerate(shapes(12000, 8)):
        dx, dw = block(lib, M, N, K, i % 2)
        pair, tile, splits = F.pair_pick(lib, dx, dw)
        if pair < 0:
            apart += 1
            continue
        for k, (family, want, p) in enumerate((("dx", pairs[pair].dx, dx), ("dw", pairs[pair].dw, dw))):
            t = F.tiles(lib, family)[tile[k]]
            assert (t.bm, t.bn, t.lds) == tuple(want) and t.occ == 2
            stages = (p.K + 63) // 64 * (2 if family == "dx" and p.a2 else 1)
            assert splits[k] == 1 or (splits[k] <= 16 and stages // splits[k] >= 8
                                      and splits[k] * p.M * p.N * 4 * (2 if p.batch else 1) <= p.part_bytes)
        assert min(splits) == 1
        taken.add((pair, splits[0] > 1, splits[1] > 1))
    assert {t[0] for t in taken} == set(range(F.PAIRS)) and apart > 500
    assert {t[1:] for t in taken} == {(False, False), (True, False), (False, True)}
    dx, dw = block(lib, 300, 512, 256, 0)
    assert F.pair_pick(lib, dx, dw)[0] >= 0
    dw.b = F.AT + 2                                                 # x that direct loads cannot take
    assert F.pair_pick(lib, dx, dw)[0] == -1
