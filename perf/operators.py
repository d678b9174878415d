"""Dense feed-forward operators as an engine, or a program that tunes one, calls them: the linear with bias, activation
and residual in its epilogue (BF16 and FP8-block weights), the gated projections of a feed-forward block (both products,
the activation and their product), and the backward passes of the two (BF16 weights).

  linear      y = act(x W^T + b) + r
  gated       h = act(min(x Wg^T, limit)) * clamp(x Wu^T, -limit, limit)
  linear_bwd  dx, dW, db of the linear from dy (its z computed again)
  gated_bwd   dx, dWg, dWu of the gated projections from dh (g and u computed again)

Sizes are those of this repository's configurations (hidden 4096, expert and shared-expert intermediate 2048, o_proj
4096x16384, q_a 1536x4096) and a generic dense block of 4096/12288.
"""
import math
import os

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda"
ACTS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}


def _case(name, op, weights, M, N, K, act="none", bias=False, residual=False, limit=0.0, pad=0):
    case = {"op": op, "weights": weights, "M": M, "N": N, "K": K, "act": act, "bias": bias, "residual": residual,
            "limit": limit, "pad": pad}
    return dict(case, name=name) if name else case


def listed():
    return [
        # one decode token: the shared-expert-sized down projection onto the residual stream
        _case("linear bf16 down M1", "linear", "bf16", 1, 4096, 2048, residual=True),
        # a speculative verify (1 token + 3 drafts): o_proj onto the residual stream
        _case("linear fp8 o_proj M4", "linear", "fp8", 4, 4096, 16384, residual=True),
        # a short prompt through a biased, activated projection of ragged width
        _case("linear bf16 bias gelu M37", "linear", "bf16", 37, 1537, 4096, act="gelu", bias=True),
        # a long prompt: the dense block's down projection onto the residual stream
        _case("linear bf16 down M4096", "linear", "bf16", 4096, 4096, 12288, residual=True),
        # one decode token through the dense block's gate and up projections
        _case("gated fp8 M1", "gated", "fp8", 1, 12288, 4096, act="silu", limit=10.0),
        # a batch of five requests through BF16 gate and up projections
        _case("gated bf16 M5", "gated", "bf16", 5, 2048, 4096, act="gelu_tanh"),
        # a prompt of no particular length through a shared expert's projections
        _case("gated fp8 M1111", "gated", "fp8", 1111, 2048, 4096, act="silu", limit=10.0),
        # the longest prompt through the dense block's projections
        _case("gated bf16 M8192", "gated", "bf16", 8192, 12288, 4096, act="silu"),
        # a small tuning batch: a biased, activated projection's gradients
        _case("linear bwd gelu M300", "linear_bwd", "bf16", 300, 2048, 1536, act="gelu", bias=True),
        # a training step's down projection
        _case("linear bwd M4096", "linear_bwd", "bf16", 4096, 4096, 12288),
        # a small tuning batch through a shared-expert-sized block
        _case("gated bwd M500", "gated_bwd", "bf16", 500, 2048, 4096, act="silu", limit=10.0),
        # a training step of the dense block
        _case("gated bwd M4096", "gated_bwd", "bf16", 4096, 12288, 4096, act="silu"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "gated", "gated", "linear_bwd", "gated_bwd"])
    weights = rng.choice(["bf16", "fp8"]) if op in ("linear", "gated") else "bf16"
    N = _log(rng, 64, 16384 if op == "linear" else 12288)
    if rng.random() < 0.6:  # most widths are whole vectors of 8, the others any number
        N = max(8, N // 8 * 8)
    K = (128 if weights == "fp8" else 64) * _log(rng, 2, 64)
    if rng.random() < 0.15:  # rows that end inside a block of 64 or 128
        K += 8 * rng.randint(1, 7)
    M = _log(rng, 1, 8192) if op in ("linear", "gated") else _log(rng, 16, 4096)
    gated = op.startswith("gated")
    act = rng.choice(["silu", "silu", "gelu_tanh", "gelu", "relu"] if gated else ["none", "none", "silu", "gelu", "relu"])
    return _case(None, op, weights, M, N, K, act=act, bias=not gated and rng.random() < 0.5,
                 residual=op == "linear" and rng.random() < 0.5, limit=rng.choice([0.0, 10.0]) if gated else 0.0,
                 # rows of x inside a wider buffer (a slice of a fused projection or a residual stream of several lanes)
                 pad=8 * rng.randint(1, 64) if rng.random() < 0.25 else 0)


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


def _weight(gen, N, K, fp8):
    """Weights of a trained layer's scale: N(0, 1/K). As FP8 blocks: codes and the scale of each 128x128 block."""
    w = torch.randn(N, K, generator=gen, device=DEV) / math.sqrt(K)
    if not fp8:
        return {"w": w.bfloat16()}
    nb, kb = -(-N // 128), -(-K // 128)
    full = torch.zeros(nb * 128, kb * 128, device=DEV)
    full[:N, :K] = w
    scale = full.view(nb, 128, kb, 128).abs().amax((1, 3)) / 448.0
    q = full.view(nb, 128, kb, 128) / scale[:, None, :, None]
    codes = q.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(nb * 128, kb * 128)[:N, :K]
    return {"codes": codes.contiguous().view(torch.uint8), "scales": scale.contiguous()}


def prepare(case, seed):
    c = case
    gen = torch.Generator(device=DEV).manual_seed(seed)
    M, N, K = c["M"], c["N"], c["K"]
    rnd = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    s = {"case": c, "x": rnd(M, K + c["pad"]).bfloat16()[:, :K]}
    # gates reach a clamp of 10 now and then, as they do in a trained layer
    spread = 4.0 if c["limit"] else 1.0
    for key in ("a", "b") if c["op"].startswith("gated") else ("a",):
        w = _weight(gen, N, K, c["weights"] == "fp8")
        s[key] = {k: v * spread if k in ("w", "scales") else v for k, v in w.items()}
    s["bias"] = rnd(N).bfloat16() if c["bias"] else None
    s["residual"] = rnd(M, N).bfloat16() if c["residual"] else None
    bf = lambda *n: torch.empty(*n, dtype=torch.bfloat16, device=DEV)  # noqa: E731
    # what a program keeps from call to call: the outputs' buffers and the backward's workspace
    if c["op"].endswith("bwd"):
        s["dy"] = rnd(M, N).bfloat16()
        s["out"] = {"dx": bf(M, K), "dw": [bf(N, K) for _ in range(2 if c["op"] == "gated_bwd" else 1)]}
        if c["bias"]:
            s["out"]["db"] = bf(N)
    else:
        s["out"] = bf(M, N)
    return s


def _p(t):
    return None if t is None else t.data_ptr()


def _own(s):
    c, lib = s["case"], _lib()
    M, N, K, act, lim = c["M"], c["N"], c["K"], ACTS[c["act"]], c["limit"]
    st, x, ldx, out, a = torch.cuda.current_stream().cuda_stream, s["x"].data_ptr(), s["x"].stride(0), s["out"], s["a"]
    if c["op"] == "linear":
        if c["weights"] == "bf16":
            rc = lib.apus_ghip_bf16_linear_ep_dev(_p(a["w"]), x, _p(s["bias"]), _p(s["residual"]), _p(out), M, N, K, ldx, 0, 0, act, st)
        else:
            rc = lib.apus_ghip_fp8blk_linear_ep_dev(_p(a["codes"]), _p(a["scales"]), x, _p(s["bias"]), _p(s["residual"]), _p(out),
                                                    M, N, K, ldx, 0, 0, act, 0, st)
    elif c["op"] == "gated":
        b = s["b"]
        if c["weights"] == "bf16":
            rc = lib.apus_ghip_bf16_gated_dev(_p(a["w"]), _p(b["w"]), x, _p(out), M, N, K, ldx, 0, act, lim, st)
        else:
            rc = lib.apus_ghip_fp8blk_gated_dev(_p(a["codes"]), _p(a["scales"]), _p(b["codes"]), _p(b["scales"]), x, _p(out),
                                                M, N, K, ldx, 0, act, lim, 0, st)
    else:
        if "ws" not in s:
            need = (lib.apus_ghip_gated_backward_ws if c["op"] == "gated_bwd" else lib.apus_ghip_linear_ep_backward_ws)(M, N, K)
            s["ws"] = torch.empty(max(need, 1), dtype=torch.uint8, device=DEV)
        ws = s["ws"]
        if c["op"] == "linear_bwd":
            rc = lib.apus_ghip_bf16_linear_ep_backward_dev(_p(a["w"]), x, _p(s["bias"]), _p(s["dy"]), _p(out["dx"]), _p(out["dw"][0]),
                                                           _p(out.get("db")), M, N, K, ldx, 0, 0, act, ws.data_ptr(), ws.numel(), st)
        else:
            rc = lib.apus_ghip_bf16_gated_backward_dev(_p(a["w"]), _p(s["b"]["w"]), x, _p(s["dy"]), _p(out["dx"]), _p(out["dw"][0]),
                                                       _p(out["dw"][1]), M, N, K, ldx, 0, 0, act, lim, ws.data_ptr(), ws.numel(), st)
    if rc:
        raise RuntimeError("%s: %s" % (c["op"], lib.apus_ghip_last_error().decode()))
    return out


def _matrix(w):
    """The weights that the operator multiplies with, in 32 bits: FP8 blocks stand for bf16(code * scale)."""
    if "w" in w:
        return w["w"].float()
    codes = w["codes"].view(torch.float8_e4m3fn).float()
    N, K = codes.shape
    scale = w["scales"].repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    return (codes * scale).bfloat16().float()


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
    c = s["case"]
    x, wa, lim = s["x"].float(), _matrix(s["a"]), c["limit"] or math.inf
    if c["op"] in ("linear", "linear_bwd"):
        z = None
        if c["op"] == "linear" or c["act"] != "none":
            z = x @ wa.t()
            if c["bias"]:
                z = z + s["bias"].float()
        if c["op"] == "linear":
            y = _act(c["act"], z)
            return (y + s["residual"].float() if c["residual"] else y).bfloat16()
        dz = s["dy"].float() if z is None else s["dy"].float() * _slope(c["act"], z)
        out = {"dx": (dz @ wa).bfloat16(), "dw": [(dz.t() @ x).bfloat16()]}
        if c["bias"]:
            out["db"] = dz.sum(0).bfloat16()
        return out
    wb = _matrix(s["b"])
    g, u = x @ wa.t(), x @ wb.t()
    gc, uc = g.clamp(max=lim), u.clamp(-lim, lim)
    if c["op"] == "gated":
        return (_act(c["act"], gc) * uc).bfloat16()
    dh = s["dy"].float()
    dg = torch.where(g <= lim, dh * uc * _slope(c["act"], gc), 0.0)
    du = torch.where(u.abs() <= lim, dh * _act(c["act"], gc), 0.0)
    return {"dx": (dg @ wa + du @ wb).bfloat16(), "dw": [(dg.t() @ x).bfloat16(), (du.t() @ x).bfloat16()]}


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    M, N, K, op = case["M"], case["N"], case["K"], case["op"]
    w = K * N * (1 if case["weights"] == "fp8" else 2)
    if op == "linear":
        return {"bytes": 2 * M * K + w + 2 * M * N * (2 if case["residual"] else 1) + (2 * N if case["bias"] else 0), "flops": 2 * M * N * K}
    if op == "gated":
        return {"bytes": 2 * M * K + 2 * w + 2 * M * N, "flops": 4 * M * N * K}
    if op == "linear_bwd":
        return {"bytes": 4 * M * K + 2 * w + 2 * M * N + (4 * N if case["bias"] else 0), "flops": (4 if case["act"] == "none" else 6) * M * N * K}
    return {"bytes": 4 * M * K + 4 * w + 2 * M * N, "flops": 12 * M * N * K}


def exact(case, seed):
    """The same from the definitions in 64 bits; derivatives by torch's own differentiation of the forward expression."""
    s = prepare(case, seed)
    x = s["x"].double()

    def wide(w):
        if "w" in w:
            return w["w"].double()
        codes, scales = w["codes"].view(torch.float8_e4m3fn).double(), w["scales"].double()
        i = torch.arange(codes.shape[0], device=DEV) // 128
        j = torch.arange(codes.shape[1], device=DEV) // 128
        # the product is rounded to 32 bits and then to bf16: both are part of the weight's definition
        return (codes * scales[i][:, j]).float().bfloat16().double()

    def act(z):
        name = case["act"]
        if name == "silu":
            return z * torch.special.expit(z)
        if name == "gelu":
            return z * torch.special.ndtr(z)
        if name == "gelu_tanh":
            return z * torch.special.expit(2.0 * math.sqrt(2.0 / math.pi) * (z + 0.044715 * z ** 3))
        return torch.relu(z) if name == "relu" else z

    ws = [wide(s[k]) for k in ("a", "b") if k in s]
    zs = [x @ w.t() for w in ws]
    if case["bias"]:
        zs = [z + s["bias"].double() for z in zs]
    grad = case["op"].endswith("bwd")
    zs = [z.requires_grad_(grad) for z in zs]
    if len(zs) == 1:
        y = act(zs[0])
        if case["residual"]:
            y = y + s["residual"].double()
    else:
        lim = case["limit"]
        y = act(zs[0].clamp(max=lim) if lim else zs[0]) * (zs[1].clamp(-lim, lim) if lim else zs[1])
    if not grad:
        return y
    ds = [t.detach() for t in torch.autograd.grad(y, zs, s["dy"].double())]
    dx = ds[0] @ ws[0]
    if len(ds) == 2:
        dx = dx + ds[1] @ ws[1]
    out = {"dx": dx, "dw": [d.t() @ x for d in ds]}
    if case["bias"]:
        out["db"] = ds[0].sum(0)
    return out
