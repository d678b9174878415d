"""The internal launchers of the products with MXFP4 weights (ghip_internal.h), so
that tests can run each kernel by itself."""
import ctypes

import ffn_forms as F
import gpu_util as G

LINEAR, GATED = F.LINEAR, F.GATED


class Prod(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in ("w", "w2", "ws", "ws2", "x", "xs")] + [("xld", ctypes.c_size_t)]
                + [(n, ctypes.c_uint32) for n in ("M", "N", "K")] + [("xt", ctypes.c_int)])


def prod(xt, M, N, K, w, ws, x, xs=None, w2=None, ws2=None, xld=0):
    return Prod(w=w, w2=w2, ws=ws, ws2=ws2, x=x, xs=xs, xld=xld or K * (4, 2, 1)[xt] // 2, M=M, N=N, K=K, xt=xt)


def tiles(lib, mode, xt):
    return lib.ghip_mx_gemm_tiles(mode, xt)


def rows(lib, mode, xt):
    return lib.ghip_mx_rows_forms(mode, xt)


def rows_fits(lib, mode, form, xt, M, N, K):
    at = 1 << 20                                                    # never read
    return lib.ghip_mx_rows_fits(mode, form, ctypes.byref(prod(xt, M, N, K, at, at, at, at, at, at)))


def launch(lib, kind, mode, form, p, ep, st=None):
    """kind: gemm or rows; the hipError_t."""
    return getattr(lib, "ghip_launch_mx_" + kind)(mode, form, ctypes.byref(p), ctypes.byref(ep), st)


def run(lib, kind, mode, form, a, w, w2, y, bias=None, res=None, act=0, limit=float("inf")):
    """a, w, w2: test_gpu_mx's Act and Mx; y, res: Mat."""
    M, N, K = y.rows, y.cols, w.values.shape[1]
    at = lambda b: None if b is None else G.vp(b).value  # noqa: E731
    x, xs = (a.mat.p.value, None) if a.type == 0 else (at(a.mx.codes), at(a.mx.scales))
    p = prod(a.type, M, N, K, at(w.codes), at(w.scales), x, xs, at(w2 and w2.codes), at(w2 and w2.scales),
             2 * a.mat.ld if a.type == 0 else 0)
    ep = F.Ep(bias=at(bias), in_=None if res is None else res.p.value, out=y.p.value, ldin=0 if res is None else res.ld, ldout=y.ld, act=act,
              limit=limit)
    return launch(lib, kind, mode, form, p, ep)
