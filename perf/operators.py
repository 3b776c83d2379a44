"""The operators around a 4-bit frozen linear layer: root-mean-square norm (with the residual's addition and 8- or 4-bit outputs) and its backward, microscaled
4-bit quantisation and its way back, the product on those operands, and a layer made of them with its input gradient.

A case is a dict: `op` names the operator, the other entries are sizes, types and options.  Plain forms are elementary torch operations in 32 bits."""
import math

import torch

own = False

BLOCK = 32            # elements that share one power-of-two scale
CHUNK = 256           # elements whose 8 scale bytes lie together
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-6


def listed():
    return [
        # decoding: one token, the norm in front of a layer; nothing but latency
        {"name": "norm token", "op": "norm", "rows": 1, "C": 1024, "dtype": "bf16", "res": True, "fmt": "e4m3"},
        # the frames of one training batch (32 clips x 8 frames x 197 tokens), norm writing the 8-bit operand of the next product
        {"name": "norm batch e4m3", "op": "norm", "rows": 50432, "C": 768, "dtype": "bf16", "res": True, "fmt": "e4m3"},
        # the fp32 parity mode on a width no vector divides
        {"name": "norm odd f32", "op": "norm", "rows": 3001, "C": 1411, "dtype": "f32", "res": False, "fmt": "same"},
        # a few frames of a wide model, 4-bit operand, read back
        {"name": "norm wide mxfp4", "op": "norm", "rows": 788, "C": 8192, "dtype": "bf16", "res": True, "fmt": "mxfp4"},
        # training: the gradient through the norm, added to the residual stream's
        {"name": "norm gradient", "op": "norm_bwd", "rows": 50432, "C": 768, "dtype": "bf16", "dy": "bf16", "dres": True},
        # loading a checkpoint: fp32 master weights to 4 bits
        {"name": "quantise weights", "op": "quant", "rows": 4096, "C": 1024, "dtype": "f32", "transpose": False},
        # the operand of a gradient product: 64 frames, quantised along the tokens
        {"name": "quantise columns", "op": "quant", "rows": 12608, "C": 768, "dtype": "bf16", "transpose": True},
        # decoding: one token through a 4-bit layer; the weights' bytes and latency
        {"name": "product token", "op": "product", "M": 1, "N": 4096, "K": 1024, "a": "e4m3", "out": "bf16", "bias": True, "res": False},
        # one frame through odd sizes
        {"name": "product ragged", "op": "product", "M": 197, "N": 1411, "K": 416, "a": "mxfp4", "out": "f32", "bias": True, "res": True},
        # the q | k | v projection of a training batch: the output's bytes
        {"name": "product wide", "op": "product", "M": 50432, "N": 2304, "K": 768, "a": "mxfp4", "out": "bf16", "bias": True, "res": False},
        # the second Linear of an MLP on 64 frames of 257 tokens: the matrix cores
        {"name": "product deep", "op": "product", "M": 16448, "N": 1024, "K": 4096, "a": "e4m3", "out": "bf16", "bias": True, "res": True},
        # training through a frozen layer: norm + product forward, then the product and the norm of the gradient
        {"name": "layer and gradient", "op": "layer", "rows": 12608, "C": 768, "N": 2304, "dtype": "bf16"},
    ]


def _spread(rng, low, high, step=1):
    """a whole number between low and high, evenly over the logarithm, a multiple of step"""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high))) / step)) * step))


def draw(rng):
    op = rng.choice(["norm", "norm", "norm_bwd", "quant", "product", "product", "product", "layer"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op in ("norm", "norm_bwd", "quant"):
        C = _spread(rng, 32, 8192, rng.choice([1, 8, 32]))
        rows = _spread(rng, 1, max(1, min(50432, 30_000_000 // C // (2 if dtype == "f32" else 1))))
        if op == "norm":
            fmt = rng.choice(["same", "e4m3", "mxfp4"])
            return {"op": op, "rows": rows, "C": C, "dtype": dtype, "res": rng.random() < 0.6, "fmt": fmt}
        if op == "norm_bwd":
            return {"op": op, "rows": rows, "C": C, "dtype": dtype, "dy": rng.choice(["bf16", "f32"]), "dres": rng.random() < 0.6}
        return {"op": op, "rows": rows, "C": C, "dtype": dtype, "transpose": rng.random() < 0.4}
    K = _spread(rng, 32, 4096, 32)
    N = _spread(rng, 16, 4096, rng.choice([1, 8, 64]))
    M = _spread(rng, 1, max(1, min(50432, 80_000_000_000 // (2 * N * K), 35_000_000 // max(N, K))))
    if op == "product":
        a = rng.choice(["mxfp4", "e4m3"])
        return {"op": op, "M": M, "N": N, "K": K, "a": a, "out": rng.choice(["bf16", "f32"]) if a == "mxfp4" else "bf16",
                "bias": rng.random() < 0.7, "res": rng.random() < 0.4}
    return {"op": op, "rows": max(1, min(M, 12608)), "C": K, "N": N, "dtype": dtype}


# ---- plain forms --------------------------------------------------------------------------------------------------------------------------------------

def _up(n, to):
    return -(-n // to) * to


def _blocks(x):
    """fp32 x [rows, K] -> (values on the 4-bit grid before scaling [rows, blocks, 32], exponents [rows, blocks])"""
    rows, K = x.shape
    x = torch.nn.functional.pad(x, (0, _up(K, BLOCK) - K)).view(rows, -1, BLOCK)
    e = (torch.frexp(x.abs().amax(-1))[1] - 3).clamp(-127, 125)              # floor(log2 a) - 2
    e = torch.where(x.abs().amax(-1) == 0, -127, e)
    v = torch.ldexp(x, -e[..., None])
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return torch.copysign((torch.round(a / step) * step).clamp(max=6.0), v), e


def _on_grid(x):
    """x rounded to 4 bits in blocks, as the fp32 values this stands for, [rows, K up to a whole block]"""
    v, e = _blocks(x)
    return torch.ldexp(v, e[..., None]).flatten(1)


def _pack(x):
    """fp32 x [rows, K] -> (codes [rows, K/2], scales [chunks, rows, 8]) in the layout the product reads"""
    v, e = _blocks(x)
    rows, nb = e.shape
    a = v.abs().flatten(1)
    code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8) | (torch.signbit(v.flatten(1)).to(torch.uint8) << 3)
    codes = code[:, 0::2] | (code[:, 1::2] << 4)
    s = torch.zeros(rows, _up(nb, 8), dtype=torch.uint8, device=x.device)
    s[:, :nb] = (e + 127).to(torch.uint8)
    return codes.contiguous(), s.view(rows, -1, 2, 4).permute(1, 0, 3, 2).reshape(-1, rows, 8).contiguous()


def _unpack(codes, scales):
    """(codes, scales) -> the fp32 values they stand for, [rows, K]"""
    rows, half = codes.shape
    code = torch.stack([codes & 15, codes >> 4], -1).view(rows, half * 2)
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    e = scales.view(-1, rows, 4, 2).permute(1, 0, 3, 2).reshape(rows, -1)[:, :half * 2 // BLOCK].to(torch.int32) - 127
    return torch.ldexp(grid[code.long()].view(rows, -1, BLOCK), e[..., None]).flatten(1)


def _plain_norm(x, w, res):
    h = x.float() + res.float() if res is not None else x.float()
    rstd = 1 / torch.sqrt(h.square().mean(-1) + EPS)
    return h, rstd, h * rstd[:, None] * w


def _plain_e4m3(y):
    a = y.abs().amax(-1)
    scale = torch.where(a > 0, a / 448, 1.0)
    inv = torch.where(a > 0, 448 / a, 1.0)
    return (y * inv[:, None]).to(torch.float8_e4m3fn), scale


def _plain_norm_bwd(h, rstd, dy, w, dres):
    g, xh = dy.float() * w, h.float() * rstd[:, None]
    dh = rstd[:, None] * (g - xh * (g * xh).mean(-1, keepdim=True))
    if dres is not None:
        dh = dh + dres.float()
    return dh.to(h.dtype), (dy.float() * xh).sum(0)


# ---- inputs -------------------------------------------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, dtype=torch.float32, std=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)

    def activations(rows, C, dtype):
        """the residual stream of a transformer: columns of very different size, some of them far above the others"""
        size = torch.exp(normal(C) * 0.7)
        return (normal(rows, C) * size).to(dtype)

    op, s = case["op"], dict(case)
    if op == "norm":
        t = TYPES[case["dtype"]]
        s |= {"x": activations(case["rows"], case["C"], t), "w": 1 + normal(case["C"], std=0.2)}
        s["r"] = activations(case["rows"], case["C"], t) if case["res"] else None
    elif op == "norm_bwd":
        t = TYPES[case["dtype"]]
        s |= {"h": activations(case["rows"], case["C"], t), "w": 1 + normal(case["C"], std=0.2), "d": normal(case["rows"], case["C"], dtype=TYPES[case["dy"]], std=1e-2)}
        s["r"] = normal(case["rows"], case["C"], dtype=t, std=1e-2) if case["dres"] else None
        s["rstd"] = 1 / torch.sqrt(s["h"].float().square().mean(-1) + EPS)
    elif op == "quant":
        s["x"] = activations(case["rows"], case["C"], TYPES[case["dtype"]]) * 0.05
    elif op == "product":
        M, N, K = case["M"], case["N"], case["K"]
        s["B"] = _pack(normal(N, K, std=K ** -0.5))
        if case["a"] == "mxfp4":
            s["A"] = _pack(normal(M, K))
        else:
            q, scale = _plain_e4m3(normal(M, K))
            s["A"] = (q.view(torch.uint8), scale)
        s["bias"] = normal(N, std=0.1) if case["bias"] else None
        s["r"] = normal(M, N, dtype=TYPES[case["out"]]) if case["res"] else None
    else:
        rows, C, N, t = case["rows"], case["C"], case["N"], TYPES[case["dtype"]]
        W = normal(N, C, std=C ** -0.5)
        s |= {"x": activations(rows, C, t), "r": activations(rows, C, t), "w": 1 + normal(C, std=0.2), "bias": normal(N, std=0.1),
              "W": _pack(W), "WT": _pack(W.t().contiguous()), "d": normal(rows, N, dtype=t, std=1e-2), "dres": normal(rows, C, dtype=t, std=1e-2)}
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------------------------------------------

def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_plain(s):
    op = s["op"]
    if op == "norm":
        h, rstd, y = _plain_norm(s["x"], s["w"], s["r"])
        out = {"rstd": rstd}
        if s["r"] is not None:
            out["h"] = h.to(s["x"].dtype)
        if s["fmt"] == "same":
            out["y"] = y.to(s["x"].dtype)
        elif s["fmt"] == "e4m3":
            out["q"], out["scale"] = _plain_e4m3(y)
        else:
            out["values"] = _on_grid(y).to(torch.bfloat16)
        return out
    if op == "norm_bwd":
        return _plain_norm_bwd(s["h"], s["rstd"], s["d"], s["w"], s["r"])
    if op == "quant":
        x = s["x"].float()
        return _on_grid(x.t() if s["transpose"] else x).to(torch.bfloat16)
    if op == "product":
        B = _unpack(*s["B"])
        c = _unpack(*s["A"]) @ B.t() if s["a"] == "mxfp4" else (s["A"][0].view(torch.float8_e4m3fn).float() @ B.t()) * s["A"][1][:, None]
        if s["bias"] is not None:
            c = c + s["bias"]
        if s["r"] is not None:
            c = c + s["r"].float()
        return c.to(TYPES[s["out"]])
    t = s["x"].dtype
    h, rstd, y = _plain_norm(s["x"], s["w"], s["r"])
    q, scale = _plain_e4m3(y)
    z = (q.float() @ _unpack(*s["W"]).t()) * scale[:, None] + s["bias"]
    dy = _on_grid(s["d"].float()) @ _unpack(*s["WT"]).t()
    dx, dw = _plain_norm_bwd(h.to(t), rstd, dy, s["w"], s["dres"])
    return {"z": z.to(torch.bfloat16), "h": h.to(t), "dx": dx, "dw": dw}


def _run_own(s):
    from dist_amd import ops
    op = s["op"]
    if op == "norm":
        rstd = torch.empty(s["x"].shape[0], dtype=torch.float32, device=s["x"].device)
        n = ops.rmsnorm(s["x"], s["w"], res=s["r"], fmt=s["fmt"], rstd=rstd, eps=EPS)
        out = {"rstd": rstd}
        if s["r"] is not None:
            out["h"] = n["h"]
        if s["fmt"] == "same":
            out["y"] = n["y"]
        elif s["fmt"] == "e4m3":
            out["q"], out["scale"] = n["q"].view(torch.float8_e4m3fn), n["scale"]
        else:
            out["values"] = ops.dequant_mxfp4(n["codes"], n["scales"])
        return out
    if op == "norm_bwd":
        return ops.rmsnorm_bwd(s["h"], s["rstd"], s["d"], s["w"], dres=s["r"])
    if op == "quant":
        return ops.dequant_mxfp4(*ops.quant_mxfp4(s["x"], transpose=s["transpose"]))
    if op == "product":
        return ops.gemm_mxfp4(s["A"], s["B"], bias=s["bias"], res=s["r"], out_dtype=TYPES[s["out"]])
    rstd = torch.empty(s["x"].shape[0], dtype=torch.float32, device=s["x"].device)
    n = ops.rmsnorm(s["x"], s["w"], res=s["r"], fmt="e4m3", rstd=rstd, eps=EPS)
    z = ops.gemm_mxfp4((n["q"], n["scale"]), s["W"], bias=s["bias"])
    dy = ops.gemm_mxfp4(ops.quant_mxfp4(s["d"]), s["WT"], out_dtype=torch.float32)
    dx, dw = ops.rmsnorm_bwd(n["h"], rstd, dy, s["w"], dres=s["dres"])
    return {"z": z, "h": n["h"], "dx": dx, "dw": dw}


# ---- bytes and operations that a pass cannot do without -----------------------------------------------------------------------------------------------

def _size(name):
    return TYPES[name].itemsize


def _four(rows, K):
    return rows * (_up(K, BLOCK) // 2 + _up(K, BLOCK) // BLOCK)


def work(case):
    op = case["op"]
    if op == "norm":
        n, e = case["rows"] * case["C"], _size(case["dtype"])
        put = {"same": n * e, "e4m3": n + 4 * case["rows"], "mxfp4": 2 * _four(case["rows"], case["C"]) + 2 * case["rows"] * _up(case["C"], BLOCK)}[case["fmt"]]
        return {"bytes": n * e * (3 if case["res"] else 1) + put + 4 * case["C"] + 4 * case["rows"], "flops": 6 * n}
    if op == "norm_bwd":
        n, e = case["rows"] * case["C"], _size(case["dtype"])
        return {"bytes": n * (e * (3 if case["dres"] else 2) + _size(case["dy"])) + 8 * case["C"] + 4 * case["rows"], "flops": 10 * n}
    if op == "quant":
        rows, K = (case["C"], case["rows"]) if case["transpose"] else (case["rows"], case["C"])
        return {"bytes": rows * K * _size(case["dtype"]) + 2 * _four(rows, K) + 2 * rows * _up(K, BLOCK), "flops": 4 * rows * K}
    if op == "product":
        M, N, K = case["M"], case["N"], case["K"]
        a = _four(M, K) if case["a"] == "mxfp4" else M * K + 4 * M
        return {"bytes": a + _four(N, K) + M * N * _size(case["out"]) * (2 if case["res"] else 1) + (4 * N if case["bias"] else 0), "flops": 2 * M * N * K}
    rows, C, N, e = case["rows"], case["C"], case["N"], _size(case["dtype"])
    return {"bytes": rows * C * e * 5 + rows * N * (e + 2) + _four(N, C) + _four(C, N) + 8 * C + 4 * N, "flops": 4 * rows * N * C}


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------------------------------------

_E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _exact_four(x):
    """nearest 4-bit values in 64 bits, [rows, whole blocks]: the border between two neighbours goes to the one with the even code"""
    rows, K = x.shape
    b = torch.zeros(rows, _up(K, BLOCK), dtype=torch.float64, device=x.device)
    b[:, :K] = x
    b = b.view(-1, BLOCK)
    top = b.abs().max(1).values
    floor = torch.floor(torch.log2(top.clamp(min=2.0 ** -200)))
    floor += (torch.exp2(floor + 1) <= top).double() - (torch.exp2(floor) > top).double()        # (log2 next to a power of two)
    unit = torch.exp2((floor - 2).clamp(-127, 125))[:, None]
    a = b.abs() / unit
    out = torch.zeros_like(a)
    for k in range(1, 8):
        border = (_E2M1[k - 1] + _E2M1[k]) / 2
        out = torch.where((a >= border) if k % 2 == 0 else (a > border), _E2M1[k], out)
    return (out * unit * torch.sign(b)).view(rows, -1)


def _exact_read(codes, scales):
    rows, half = codes.shape
    c = codes.long()
    level = torch.tensor(_E2M1, dtype=torch.float64, device=codes.device)
    out = torch.empty(rows, 2 * half, dtype=torch.float64, device=codes.device)
    for k, n in enumerate((c % 16, c // 16)):
        out[:, k::2] = level[n % 8] * (1 - 2 * (n // 8).double())
    for block in range(2 * half // BLOCK):
        chunk, within = divmod(block, 8)
        e = scales[chunk, :, 2 * (within % 4) + within // 4].double() - 127
        out[:, block * BLOCK:(block + 1) * BLOCK] *= torch.exp2(e)[:, None]
    return out


def _exact_e4m3(y):
    a = y.abs().max(1).values
    scale = torch.where(a > 0, a / 448, torch.ones_like(a))
    v = y / scale[:, None]
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(v / step) * step).clamp(-448, 448), scale


def _exact_norm(x, w, r):
    h = x.double() if r is None else x.double() + r.double()
    rstd = (h.pow(2).sum(1) / h.shape[1] + EPS).pow(-0.5)
    return h, rstd, rstd[:, None] * h * w.double()


def _exact_norm_bwd(h, rstd, dy, w, dres):
    n, d = h.double() * rstd.double()[:, None], dy.double()
    inner = (d * w.double() * n).sum(1, keepdim=True) / h.shape[1]
    dh = (d * w.double() - n * inner) * rstd.double()[:, None]
    return dh if dres is None else dh + dres.double(), (d * n).sum(0)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        h, rstd, y = _exact_norm(s["x"], s["w"], s["r"])
        out = {"rstd": rstd}
        if s["r"] is not None:
            out["h"] = h
        if case["fmt"] == "same":
            out["y"] = y
        elif case["fmt"] == "e4m3":
            out["q"], out["scale"] = _exact_e4m3(y)
        else:
            out["values"] = _exact_four(y)
        return out
    if op == "norm_bwd":
        return _exact_norm_bwd(s["h"], s["rstd"], s["d"], s["w"], s["r"])
    if op == "quant":
        x = s["x"].double()
        return _exact_four(x.t() if case["transpose"] else x)
    if op == "product":
        A = _exact_read(*s["A"]) if case["a"] == "mxfp4" else s["A"][0].view(torch.float8_e4m3fn).double() * s["A"][1].double()[:, None]
        c = torch.mm(A, _exact_read(*s["B"]).t().contiguous())
        if s["bias"] is not None:
            c += s["bias"].double()
        if s["r"] is not None:
            c += s["r"].double()
        return c
    h, rstd, y = _exact_norm(s["x"], s["w"], s["r"])
    q, scale = _exact_e4m3(y)
    z = torch.mm(q * scale[:, None], _exact_read(*s["W"]).t().contiguous()) + s["bias"].double()
    dy = torch.mm(_exact_four(s["d"].double()), _exact_read(*s["WT"]).t().contiguous())
    dx, dw = _exact_norm_bwd(h.to(s["x"].dtype), rstd, dy, s["w"], s["dres"])
    return {"z": z, "h": h, "dx": dx, "dw": dw}
