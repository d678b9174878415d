"""The norm in front of a projection and projections with 4-bit weights, as an engine, or a program that tunes one, calls
them: the root-mean-square norm with the residual's addition (BF16 or MXFP8 out) and its gradient, microscaled
quantization and back, and the linear and gated projections with MXFP4 weights and BF16, MXFP8 or MXFP4 activations.

  norm        s = bf16(x + r), y = s / sqrt(mean(s^2) + eps) * gamma
  norm_bwd    dx = rstd (gamma dy - s rstd^2 mean(gamma dy s)) + ds, dgamma = sum over the rows of dy s rstd
  mx          per 32 values of a row: the smallest power of two at which none is past the type's largest value, and
              the values over it, rounded to the type (ties to even)
  linear      y = act(x W^T + b) + r            W in MXFP4
  gated       h = act(min(x Wg^T, limit)) * clamp(x Wu^T, -limit, limit)
  linear_bwd  dx (and db) through frozen MXFP4 weights
  gated_bwd   dx through frozen MXFP4 weights

MXFP4 is E2M1 (two codes a byte, the lower nibble first), MXFP8 E4M3, each with an E8M0 scale (2^(byte - 127)) for 32
values along k; rows of scales are whole words. Sizes are those of this repository's configurations (hidden 4096, shared
expert 2048, q_a 1536) and a generic dense block of 4096/12288.
"""
import math
import os

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda"
ACTS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}
TYPES = {"bf16": 0, "mxfp8": 1, "mxfp4": 2}
EPS = 1e-5
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _norm(name, op, M, D, out="bf16", residual=False, pad=0):
    case = {"op": op, "M": M, "D": D, "out": out, "residual": residual, "pad": pad}
    return dict(case, name=name) if name else case


def _mx(name, R, K, type, back):
    """back: read again, which is also how codes of 4 bits are returned as what they stand for."""
    case = {"op": "mx", "R": R, "K": K, "type": type, "back": back}
    return dict(case, name=name) if name else case


def _prod(name, op, x, M, N, K, act="none", bias=False, residual=False, limit=0.0, pad=0):
    case = {"op": op, "x": x, "M": M, "N": N, "K": K, "act": act, "bias": bias, "residual": residual, "limit": limit, "pad": pad}
    return dict(case, name=name) if name else case


def listed():
    return [
        # one decode token enters a sublayer: the residual's addition and the norm
        _norm("norm bf16 M1", "norm", 1, 4096, residual=True),
        # the longest prompt enters a block whose projections take 8-bit activations
        _norm("norm mxfp8 M8192", "norm", 8192, 4096, out="mxfp8", residual=True),
        # a small tuning batch through the norm of a low-rank projection
        _norm("norm bwd M300", "norm_bwd", 300, 1536),
        # a training step's norm, the stream's own gradient added
        _norm("norm bwd M8192", "norm_bwd", 8192, 4096, residual=True),
        # a dense block's weights laid out in 4 bits and read back, as a tuning step does to see what they stand for
        _mx("mx fp4 weights", 12288, 4096, "mxfp4", True),
        # a prompt of no particular length: activations between two projections to 8 bits
        _mx("mx fp8 M1111", 1111, 2048, "mxfp8", False),
        # one decode token: the dense block's down projection onto the residual stream
        _prod("linear bf16 M1", "linear", "bf16", 1, 4096, 12288, residual=True),
        # a short prompt through a biased, activated projection of ragged width
        _prod("linear mxfp8 M300", "linear", "mxfp8", 300, 1537, 4096, act="gelu", bias=True),
        # a long prompt, both operands in 4 bits: the down projection onto the residual stream
        _prod("linear mxfp4 M4096", "linear", "mxfp4", 4096, 4096, 12288, residual=True),
        # a small tuning batch: the gradient through a frozen, activated projection
        _prod("linear bwd M500", "linear_bwd", "bf16", 500, 2048, 4096, act="silu", bias=True),
        # a batch of five requests through the dense block's gate and up projections
        _prod("gated bf16 M5", "gated", "bf16", 5, 12288, 4096, act="silu", limit=10.0),
        # the longest prompt through the same, its activations from the norm in 8 bits
        _prod("gated mxfp8 M8192", "gated", "mxfp8", 8192, 12288, 4096, act="silu", limit=10.0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "norm_bwd", "mx", "linear", "linear", "linear", "gated", "gated", "linear_bwd", "gated_bwd"])
    if op.startswith("norm"):
        D = _log(rng, 64, 16384)
        out = rng.choice(["bf16", "mxfp8"]) if op == "norm" else "bf16"
        if out == "mxfp8":
            D = max(64, D // 32 * 32)
        elif rng.random() < 0.6:  # most widths are whole vectors of 8, the others any number
            D = max(64, D // 8 * 8)
        return _norm(None, op, min(_log(rng, 1, 8192), 8192 * 4096 // D), D, out=out, residual=rng.random() < 0.6,
                     # rows inside a wider buffer
                     pad=rng.randint(1, 300) if rng.random() < 0.25 else 0)
    if op == "mx":
        K = 32 * _log(rng, 1, 384)
        type = rng.choice(["mxfp8", "mxfp4"])
        return _mx(None, min(_log(rng, 1, 12288), 12288 * 4096 // K), K, type, type == "mxfp4" or rng.random() < 0.5)
    gated, bwd = op.startswith("gated"), op.endswith("bwd")
    N = _log(rng, 64, 12288 if gated else 16384)
    if rng.random() < 0.6:
        N = max(64, N // 8 * 8)
    K = 64 * _log(rng, 1, 256)
    if rng.random() < 0.25:  # rows that end inside a step of 64
        K += 32
    most = 8192 * 12288 * 4096 * 4 // (N * K * (2 if op == "linear" else 8 if op == "gated_bwd" else 4))
    return _prod(None, op, "bf16" if bwd else rng.choice(["bf16", "mxfp8", "mxfp4"]), min(_log(rng, 16 if bwd else 1, 4096 if bwd else 8192), most), N, K,
                 act=rng.choice(["silu", "silu", "gelu_tanh", "gelu", "relu"] if gated else ["none", "none", "silu", "gelu", "relu"]),
                 bias=not gated and rng.random() < 0.5, residual=op == "linear" and rng.random() < 0.5,
                 limit=rng.choice([0.0, 10.0]) if gated else 0.0, pad=8 * rng.randint(1, 64) if rng.random() < 0.2 else 0)


def _lib():
    """The framework's library, loaded once a process (it then uses the HIP runtime that torch has loaded)."""
    import importlib.util
    import sys
    if "apus_ghip" not in sys.modules:
        at = os.path.join(ROOT, "apus-glm5.3-flash_amd")
        spec = importlib.util.spec_from_file_location("apus_ghip", os.path.join(at, "__init__.py"), submodule_search_locations=[at])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["apus_ghip"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["apus_ghip"].load()


def _ld(K):
    """Bytes of a row of scales: one for 32 values, whole words."""
    return (K // 32 + 3) // 4 * 4


def _quantize(v, type):
    """Codes [R, K] as the values they stand for before scaling, their numbers, and exponents [R, K/32]; v in 32 bits."""
    b = v.unflatten(1, (-1, 32))
    m, e = torch.frexp(b.abs().amax(2))
    top, at = (0.875, 9) if type == "mxfp8" else (0.75, 3)  # 448 = 0.875 * 2^9, 6 = 0.75 * 2^3
    e = torch.where(m > 0, e - at + (m > top), -127).clamp(-127, 127)
    q = torch.ldexp(b, -e[..., None]).flatten(1)
    if type == "mxfp8":
        return q.to(torch.float8_e4m3fn), e
    a = q.abs()
    n = (a > 0.25).to(torch.uint8)
    for over in (a >= 0.75, a > 1.25, a >= 1.75, a > 2.5, a >= 3.5, a > 5.0):  # ties to the even code
        n += over
    return n + 8 * torch.signbit(q).to(torch.uint8), e


def _pack(v, type):
    """The codes and scales that a program holds."""
    q, e = _quantize(v, type)
    scales = torch.zeros(v.shape[0], _ld(v.shape[1]), dtype=torch.uint8, device=DEV)
    scales[:, : e.shape[1]] = (e + 127).to(torch.uint8)
    codes = q.view(torch.uint8) if type == "mxfp8" else q[:, 0::2] | q[:, 1::2] << 4
    return {"codes": codes.contiguous(), "scales": scales, "type": type}


def _values(q, dtype=torch.float32):
    """What codes and scales stand for."""
    if q["type"] == "mxfp8":
        v = q["codes"].view(torch.float8_e4m3fn).to(dtype)
    else:
        c = torch.stack([q["codes"] & 15, q["codes"] >> 4], 2).flatten(1).int()
        v = torch.tensor(E2M1, dtype=dtype, device=DEV)[c & 7] * (1 - 2 * (c >> 3)).to(dtype)
    e = q["scales"][:, : v.shape[1] // 32].int() - 127
    return (v.unflatten(1, (-1, 32)) * torch.pow(torch.tensor(2.0, dtype=dtype, device=DEV), e)[..., None]).flatten(1)


def prepare(case, seed):
    c = case
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    bf = lambda *n: torch.empty(*n, dtype=torch.bfloat16, device=DEV)  # noqa: E731
    by = lambda *n: torch.empty(*n, dtype=torch.uint8, device=DEV)  # noqa: E731
    s = {"case": c}

    def acts(M, K, pad=0):
        """Activations: a few channels are ten times as large as the others."""
        loud = 1.0 + 9.0 * (torch.rand(K + pad, generator=gen, device=DEV) < 0.01)
        return (rnd(M, K + pad) * loud).bfloat16()[:, :K]

    if c["op"].startswith("norm"):
        M, D = c["M"], c["D"]
        s["x"] = acts(M, D, c["pad"])
        s["gamma"] = (1.0 + 0.2 * rnd(D)).bfloat16()
        s["residual"] = rnd(M, D).bfloat16() if c["residual"] else None
        if c["op"] == "norm":
            s["out"] = {"sum": bf(M, D)} if c["residual"] else {}
            s["out"] |= {"codes": by(M, D), "scales": by(M, _ld(D))} if c["out"] == "mxfp8" else {"y": bf(M, D)}
        else:
            s["dy"] = rnd(M, D).bfloat16()
            s["rstd"] = torch.rsqrt(s["x"].float().square().mean(1) + EPS)
            s["out"] = {"dx": bf(M, D), "dgamma": bf(D)}
        return s
    if c["op"] == "mx":
        R, K = c["R"], c["K"]
        s["x"] = acts(R, K) if c["type"] == "mxfp8" else (rnd(R, K) / math.sqrt(K)).bfloat16()
        s["out"] = {"codes": by(R, K if c["type"] == "mxfp8" else K // 2), "scales": by(R, _ld(K))}
        if c["back"]:
            s["back"] = bf(R, K)
        return s
    M, N, K = c["M"], c["N"], c["K"]
    x = acts(M, K, c["pad"] if c["x"] == "bf16" else 0)
    s["x"] = x if c["x"] == "bf16" else _pack(x.float(), c["x"])
    # gates reach a clamp of 10 now and then, as they do in a trained layer
    spread = (4.0 if c["limit"] else 1.0) / math.sqrt(K)
    for key in ("a", "b") if c["op"].startswith("gated") else ("a",):
        s[key] = _pack((rnd(N, K) * spread).bfloat16().float(), "mxfp4")
    s["bias"] = rnd(N).bfloat16() if c["bias"] else None
    s["residual"] = rnd(M, N).bfloat16() if c["residual"] else None
    if c["op"].endswith("bwd"):
        s["dy"] = rnd(M, N).bfloat16()
        s["out"] = {"dx": bf(M, K)}
        if c["bias"]:
            s["out"]["db"] = bf(N)
    else:
        s["out"] = bf(M, N)
    return s


def _p(t):
    return None if t is None else t.data_ptr()


def _workspace(s, need):
    """Kept from call to call."""
    if "ws" not in s:
        s["ws"] = torch.empty(max(need, 1), dtype=torch.uint8, device=DEV)
    return s["ws"].data_ptr(), s["ws"].numel()


def _own(s):
    c, lib, out = s["case"], _lib(), s["out"]
    st, op = torch.cuda.current_stream().cuda_stream, c["op"]
    result = out
    if op == "norm":
        M, D, x = c["M"], c["D"], s["x"]
        rc = lib.apus_ghip_rmsnorm_dev(x.data_ptr(), _p(s["residual"]), s["gamma"].data_ptr(), _p(out.get("sum")), _p(out.get("y")),
                                       _p(out.get("codes")), _p(out.get("scales")), None, M, D, x.stride(0), 0, 0, 0, EPS, st)
        if "codes" in out:
            result = _as_floats(out, D)
    elif op == "norm_bwd":
        M, D, x = c["M"], c["D"], s["x"]
        ws, n = _workspace(s, lib.apus_ghip_rmsnorm_backward_ws(M, D))
        rc = lib.apus_ghip_rmsnorm_backward_dev(x.data_ptr(), s["gamma"].data_ptr(), s["rstd"].data_ptr(), s["dy"].data_ptr(), _p(s["residual"]),
                                                out["dx"].data_ptr(), out["dgamma"].data_ptr(), M, D, x.stride(0), 0, 0, 0, EPS, ws, n, st)
    elif op == "mx":
        R, K, t, codes, scales = c["R"], c["K"], TYPES[c["type"]], out["codes"].data_ptr(), out["scales"].data_ptr()
        rc = lib.apus_ghip_mx_quantize_dev(t, s["x"].data_ptr(), codes, scales, R, K, 0, st)
        if c["back"]:
            rc = rc or lib.apus_ghip_mx_dequant_dev(t, codes, scales, s["back"].data_ptr(), R, K, 0, st)
            result = s["back"]
        else:
            result = _as_floats(out, K)
    else:
        M, N, K, act, lim, a, x = c["M"], c["N"], c["K"], ACTS[c["act"]], c["limit"], s["a"], s["x"]
        wide = c["x"] == "bf16"
        xs, xp, ldx = (None, x.data_ptr(), x.stride(0)) if wide else (x["scales"].data_ptr(), x["codes"].data_ptr(), 0)
        w, ws_ = a["codes"].data_ptr(), a["scales"].data_ptr()
        if op.startswith("gated"):
            b, bs = s["b"]["codes"].data_ptr(), s["b"]["scales"].data_ptr()
        if op == "linear":
            rc = lib.apus_ghip_mxfp4_linear_dev(w, ws_, TYPES[c["x"]], xp, xs, _p(s["bias"]), _p(s["residual"]), out.data_ptr(), M, N, K, ldx, 0, 0, act, st)
        elif op == "gated":
            rc = lib.apus_ghip_mxfp4_gated_dev(w, ws_, b, bs, TYPES[c["x"]], xp, xs, out.data_ptr(), M, N, K, ldx, 0, act, lim, st)
        elif op == "linear_bwd":
            ws, n = _workspace(s, lib.apus_ghip_mxfp4_linear_backward_ws(M, N, K))
            rc = lib.apus_ghip_mxfp4_linear_backward_dev(w, ws_, xp, _p(s["bias"]), s["dy"].data_ptr(), out["dx"].data_ptr(), _p(out.get("db")),
                                                         M, N, K, ldx, 0, 0, act, ws, n, st)
        else:
            ws, n = _workspace(s, lib.apus_ghip_mxfp4_gated_backward_ws(M, N, K))
            rc = lib.apus_ghip_mxfp4_gated_backward_dev(w, ws_, b, bs, xp, s["dy"].data_ptr(), out["dx"].data_ptr(), M, N, K, ldx, 0, 0, act, lim, ws, n, st)
    if rc:
        raise RuntimeError("%s: %s" % (op, lib.apus_ghip_last_error().decode()))
    return result


def _as_floats(out, K):
    """8-bit codes and scales as the values they stand for."""
    more = {"scales": out["scales"][:, : K // 32].view(torch.float8_e8m0fnu), "codes": out["codes"].view(torch.float8_e4m3fn)}
    return dict(out, **more)


def _mxfp8(v):
    q, e = _quantize(v, "mxfp8")
    return {"codes": q, "scales": (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)}


def _act(name, z):
    if name == "relu":
        return z.clamp(min=0.0)
    if name == "silu":
        return z / (1.0 + torch.exp(-z))
    if name == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    return z


def _slope(name, z):
    if name == "relu":
        return (z > 0.0).float()
    if name == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return s * (1.0 + z * (1.0 - s))
    if name == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2.0 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * c * (1.0 + 3.0 * 0.044715 * z * z)
    return torch.ones_like(z)


def _plain(s):
    c, op = s["case"], s["case"]["op"]
    if op == "norm":
        out = {}
        v = s["x"].float()
        if c["residual"]:
            out["sum"] = (v + s["residual"].float()).bfloat16()
            v = out["sum"].float()
        y = v * torch.rsqrt(v.square().mean(1, keepdim=True) + EPS) * s["gamma"].float()
        return dict(out, **(_mxfp8(y) if c["out"] == "mxfp8" else {"y": y.bfloat16()}))
    if op == "norm_bwd":
        v, r, dy = s["x"].float(), s["rstd"][:, None], s["dy"].float()
        n, g = v * r, dy * s["gamma"].float()
        dx = r * (g - n * (g * n).mean(1, keepdim=True))
        return {"dx": (dx + s["residual"].float() if c["residual"] else dx).bfloat16(), "dgamma": (dy * n).sum(0).bfloat16()}
    if op == "mx":
        v = s["x"].float()
        return _values(_pack(v, c["type"])).bfloat16() if c["back"] else _mxfp8(v)
    x = s["x"].float() if c["x"] == "bf16" else _values(s["x"])
    wa, lim = _values(s["a"]), c["limit"] or math.inf
    if op.startswith("linear"):
        z = None
        if op == "linear" or c["act"] != "none":
            z = x @ wa.t()
            if c["bias"]:
                z = z + s["bias"].float()
        if op == "linear":
            y = _act(c["act"], z)
            return (y + s["residual"].float() if c["residual"] else y).bfloat16()
        dz = s["dy"].float() if z is None else s["dy"].float() * _slope(c["act"], z)
        out = {"dx": (dz @ wa).bfloat16()}
        if c["bias"]:
            out["db"] = dz.sum(0).bfloat16()
        return out
    wb = _values(s["b"])
    g, u = x @ wa.t(), x @ wb.t()
    gc, uc = g.clamp(max=lim), u.clamp(-lim, lim)
    if op == "gated":
        return (_act(c["act"], gc) * uc).bfloat16()
    dh = s["dy"].float()
    dg = torch.where(g <= lim, dh * uc * _slope(c["act"], gc), 0.0)
    du = torch.where(u.abs() <= lim, dh * _act(c["act"], gc), 0.0)
    return {"dx": (dg @ wa + du @ wb).bfloat16()}


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    c, op = case, case["op"]
    if op == "norm":
        n = c["M"] * c["D"]
        return {"bytes": 2 * n * (3 if c["residual"] else 1) + (n + n // 32 if c["out"] == "mxfp8" else 2 * n) + 2 * c["D"], "flops": 5 * n}
    if op == "norm_bwd":
        n = c["M"] * c["D"]
        return {"bytes": 2 * n * (4 if c["residual"] else 3) + 4 * c["M"] + 4 * c["D"], "flops": 12 * n}
    if op == "mx":
        n = c["R"] * c["K"]
        one = n * (32 if c["type"] == "mxfp8" else 16) // 32 + n // 32
        return {"bytes": 2 * n + (2 * one + 2 * n if c["back"] else one), "flops": 4 * n}
    M, N, K = c["M"], c["N"], c["K"]
    w, x = N * K * 17 // 32, M * K * {"bf16": 64, "mxfp8": 33, "mxfp4": 17}[c["x"]] // 32
    if op == "linear":
        return {"bytes": x + w + 2 * M * N * (2 if c["residual"] else 1) + (2 * N if c["bias"] else 0), "flops": 2 * M * N * K}
    if op == "gated":
        return {"bytes": x + 2 * w + 2 * M * N, "flops": 4 * M * N * K}
    if op == "linear_bwd":
        return {"bytes": (x if c["act"] != "none" else 0) + 2 * M * K + w + 2 * M * N + (4 * N if c["bias"] else 0), "flops": (2 if c["act"] == "none" else 4) * M * N * K}
    return {"bytes": x + 2 * M * K + 2 * w + 2 * M * N, "flops": 8 * M * N * K}


def exact(case, seed):
    """The same from the definitions in 64 bits; derivatives by torch's own differentiation of the forward expression."""
    s = prepare(case, seed)
    op = case["op"]
    f64 = torch.float64

    def mx(v, type):
        """Codes and scales as values: the grid of each exponent, searched for the nearest number."""
        b = v.reshape(v.shape[0], -1, 32)
        most, mant, low = (448.0, 3, -6) if type == "mxfp8" else (6.0, 1, 0)
        amax = b.abs().max(2).values
        e = torch.ceil(torch.log2(amax.clamp(min=2.0 ** -140) / most))
        e = torch.where(amax > most * torch.exp2(e), e + 1, e)  # log2 next to a whole number
        e = torch.where(amax <= most * torch.exp2(e - 1), e - 1, e).clamp(-127, 127)
        q = b / torch.exp2(e)[..., None]
        # the spacing of the type's numbers around q
        at = torch.floor(torch.log2(q.abs().clamp(min=2.0 ** low)))
        at = torch.where(torch.exp2(at) > q.abs(), at - 1, at).clamp(min=low)
        step = torch.exp2(at - mant)
        return (torch.round(q / step) * step).reshape(v.shape), torch.exp2(e)

    if op == "norm":
        out, v = {}, s["x"].to(f64)
        if case["residual"]:
            v = (v + s["residual"].to(f64)).bfloat16().to(f64)  # rounded by its definition
            out["sum"] = v
        y = v / torch.sqrt((v * v).sum(1, keepdim=True) / case["D"] + EPS) * s["gamma"].to(f64)
        if case["out"] == "bf16":
            return dict(out, y=y)
        codes, scales = mx(y, "mxfp8")
        return dict(out, codes=codes, scales=scales)
    if op == "norm_bwd":
        v, g = s["x"].to(f64).requires_grad_(), s["gamma"].to(f64).requires_grad_()
        y = v / torch.sqrt(v.square().mean(1, keepdim=True) + EPS) * g
        dx, dg = torch.autograd.grad(y, (v, g), s["dy"].to(f64))
        return {"dx": dx + s["residual"].to(f64) if case["residual"] else dx, "dgamma": dg}
    if op == "mx":
        codes, scales = mx(s["x"].to(f64), case["type"])
        if case["back"]:
            return (codes.unflatten(1, (-1, 32)) * scales[..., None]).flatten(1)
        return {"codes": codes, "scales": scales}

    def act(z):
        name = case["act"]
        if name == "silu":
            return z * torch.special.expit(z)
        if name == "gelu":
            return z * torch.special.ndtr(z)
        if name == "gelu_tanh":
            return z * torch.special.expit(2.0 * math.sqrt(2.0 / math.pi) * (z + 0.044715 * z ** 3))
        return torch.relu(z) if name == "relu" else z

    x = s["x"].to(f64) if case["x"] == "bf16" else _values(s["x"], f64)
    ws = [_values(s[k], f64) for k in ("a", "b") if k in s]
    zs = [x @ w.t() for w in ws]
    if case["bias"]:
        zs = [z + s["bias"].to(f64) for z in zs]
    grad = op.endswith("bwd")
    zs = [z.requires_grad_(grad) for z in zs]
    if len(zs) == 1:
        y = act(zs[0])
        if case["residual"]:
            y = y + s["residual"].to(f64)
    else:
        lim = case["limit"]
        y = act(zs[0].clamp(max=lim) if lim else zs[0]) * (zs[1].clamp(-lim, lim) if lim else zs[1])
    if not grad:
        return y
    ds = [t.detach() for t in torch.autograd.grad(y, zs, s["dy"].to(f64))]
    dx = ds[0] @ ws[0]
    if len(ds) == 2:
        dx = dx + ds[1] @ ws[1]
    out = {"dx": dx}
    if case["bias"]:
        out["db"] = ds[0].sum(0)
    return out
