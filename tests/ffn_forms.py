"""The internal launchers of the dense feed-forward products (ghip_internal.h),
so that tests can ask which kernel a shape takes and run each one by itself."""
import ctypes

STORE, LINEAR, GATED, DLINEAR, DGATED = range(5)
NCU = 256


class Prod(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in ("a", "a2", "b", "b2", "s", "s2")]
                + [(n, ctypes.c_size_t) for n in ("ars", "aks", "brs", "bks")]
                + [(n, ctypes.c_uint32) for n in ("M", "N", "K")]
                + [(n, ctypes.c_int) for n in ("exact", "batch", "apad")]
                + [("part", ctypes.c_void_p), ("part_bytes", ctypes.c_size_t), ("splits", ctypes.c_uint32)])


class Ep(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in ("bias", "in_", "out", "out2")]
                + [("ldin", ctypes.c_size_t), ("ldout", ctypes.c_size_t), ("act", ctypes.c_int), ("limit", ctypes.c_float),
                   ("pad", ctypes.c_int)])


class Tile(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_uint32) for n in ("bm", "bn", "occ")] + [(n, ctypes.c_float) for n in ("low", "mid", "full", "over")]
                + [("lds", ctypes.c_uint32), ("kern", ctypes.c_void_p), ("launch", ctypes.c_void_p)])


# name: mode, weights (0 bf16, 1 FP8, 2 FP8 with NaN codes), A and B with k as the slow index
FAMILIES = {
    "linear": (LINEAR, 0, 0, 0), "linear fp8": (LINEAR, 1, 0, 0), "linear fp8 exact": (LINEAR, 2, 0, 0),
    "gated": (GATED, 0, 0, 0), "gated fp8": (GATED, 1, 0, 0), "gated fp8 exact": (GATED, 2, 0, 0),
    "dlinear": (DLINEAR, 0, 0, 0), "dgated": (DGATED, 0, 0, 0), "dx": (STORE, 0, 0, 1), "dw": (STORE, 0, 1, 1),
}
ROW_FORMS = {"linear": 8, "dlinear": 8, "gated": 6, "dgated": 6, "linear fp8": 13, "linear fp8 exact": 13, "gated fp8": 10,
             "gated fp8 exact": 10}
ROWS = [f for f, v in FAMILIES.items() if v[0] != STORE]
AT = 1 << 20                                                        # an aligned address, never read on the CPU


def tiles(lib, family):
    mode, w8, slow_a, _ = FAMILIES[family]
    n = ctypes.c_int()
    if mode in (LINEAR, GATED):
        f, arg = lib.ghip_ffn_forward_tiles, w8
    else:
        f, arg = lib.ghip_ffn_backward_tiles, slow_a
    f.restype = ctypes.POINTER(Tile)
    t = f(mode, arg, ctypes.byref(n))
    return [t[i] for i in range(n.value)]


def prod(family, M, N, K, a=AT, b=AT, a2=None, b2=None, s=None, s2=None, lda=0, ldb=0, **more):
    """The product of M x N outputs over K; lda, ldb: of the operands as they lie in memory."""
    mode, w8, slow_a, slow_b = FAMILIES[family]
    lda, ldb = lda or (M if slow_a else K), ldb or (N if slow_b else K)
    if w8 and s is None:
        s = s2 = AT
    if mode in (GATED, DGATED) and b2 is None:
        b2 = AT
    return Prod(a=a, a2=a2, b=b, b2=b2, s=s, s2=s2, ars=1 if slow_a else lda, aks=lda if slow_a else 1,
                brs=1 if slow_b else ldb, bks=ldb if slow_b else 1, M=M, N=N, K=K, exact=w8 == 2, **more)


def gemm_fits(lib, family, p):
    return lib.ghip_ffn_gemm_fits(FAMILIES[family][0], ctypes.byref(p))


def gemm_pick(lib, family, p):
    us, splits = ctypes.c_float(), ctypes.c_uint32(1)
    t = lib.ghip_ffn_gemm_pick(FAMILIES[family][0], ctypes.byref(p), ctypes.c_uint32(NCU), ctypes.byref(us), ctypes.byref(splits))
    return t, splits.value, us.value


def rows_fits(lib, family, p):
    return lib.ghip_ffn_rows_fits(FAMILIES[family][0], ctypes.byref(p))


def rows_pick(lib, family, p):
    us = ctypes.c_float()
    return lib.ghip_ffn_rows_pick(FAMILIES[family][0], ctypes.byref(p), ctypes.c_uint32(NCU), ctypes.byref(us)), us.value


def route(lib, family, p):
    """("rows", form), ("tile", tile, splits) or ("any",): ghip_launch_ffn's choice."""
    t, r = (None, 1, 1e30), (None, 1e30)
    if gemm_fits(lib, family, p):
        t = gemm_pick(lib, family, p)
    if rows_fits(lib, family, p):
        r = rows_pick(lib, family, p)
    if r[0] is not None and r[1] <= t[2]:
        return "rows", r[0]
    return ("tile", t[0], t[1]) if t[0] is not None and t[0] >= 0 else ("any",)


def part_bytes(lib, M, N, K):
    lib.ghip_ffn_part_bytes.restype = ctypes.c_size_t
    return lib.ghip_ffn_part_bytes(*(ctypes.c_size_t(v) for v in (M, N, K)))


class Sum(ctypes.Structure):
    _fields_ = [("dz", ctypes.c_void_p)] + [(n, ctypes.c_size_t) for n in ("ld", "M", "N")] + [("out", ctypes.c_void_p)]


class Pair(ctypes.Structure):
    _fields_ = [("dx", ctypes.c_uint32 * 3), ("dw", ctypes.c_uint32 * 3), ("kern", ctypes.c_void_p),
                ("launch", ctypes.CFUNCTYPE(None, *[ctypes.c_void_p] * 8))]


PAIRS = 4


def pairs(lib):
    n = ctypes.c_int()
    lib.ghip_ffn_pairs.restype = ctypes.POINTER(Pair)
    t = lib.ghip_ffn_pairs(ctypes.byref(n))
    return [t[i] for i in range(n.value)]


def pair_pick(lib, dx, dw):
    """(pair, tiles, splits) of dx and dW in one launch; pair -1: two launches."""
    tile, splits = (ctypes.c_int * 2)(), (ctypes.c_uint32 * 2)()
    i = lib.ghip_ffn_pair_pick(ctypes.byref(dx), ctypes.byref(dw), ctypes.c_uint32(NCU), tile, splits)
    return i, list(tile), list(splits)
