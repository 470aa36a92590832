"""Cases of the low-precision operators: the RMS norm and the cast that write 8-bit operands, the 8-bit GEMM that
multiplies them, and the 4-bit matrix-vector product.

An 8-bit operand is a pitched float8_e4m3fn matrix with one float32 scale per row; it stands for q * scale[:, None].
A 4-bit matrix is a pitched uint8 matrix, two weights per byte (the even column in the low nibble), with one float16
scale and optionally one uint8 zero point per `group` columns of a row; it stands for (q - zero) * scale, where zero
is 8 when there are no zero points.
"""
import math

import torch

own = False

DEV = "cuda:0"
E4M3 = torch.float8_e4m3fn
TYPES = {"f16": torch.float16, "f32": torch.float32, "e4m3": E4M3}
EPS = 1e-6


def listed():
    return [
        # one new token through the norm in front of a quantised linear layer: pure latency
        {"name": "norm_1x4096", "op": "rmsnorm_q8", "rows": 1, "cols": 4096, "type": "f16", "residual": True},
        # the same norm over a whole prompt batch: the large, bandwidth-bound end
        {"name": "norm_8192x4096", "op": "rmsnorm_q8", "rows": 8192, "cols": 4096, "type": "f16", "residual": True},
        # float32 stream, odd row length (rows not 16-byte aligned), first layer of a stack: nothing to add
        {"name": "norm_2053x3001_f32", "op": "rmsnorm_q8", "rows": 2053, "cols": 3001, "type": "f32", "residual": False},
        # activations between two linear layers of a wide block become 8-bit operands
        {"name": "cast_4096x16384", "op": "cast_q8", "rows": 4096, "cols": 16384, "type": "f16"},
        # an odd-sized float32 weight matrix is laid out as an 8-bit operand
        {"name": "cast_515x4099_f32", "op": "cast_q8", "rows": 515, "cols": 4099, "type": "f32"},
        # a decoding batch of 16 tokens through one linear layer: bound by reading the weights
        {"name": "gemm_16x4096x4096", "op": "gemm_q8", "M": 16, "N": 4096, "K": 4096, "type": "f16", "c": False},
        # a chunk of a prompt: neither tall nor flat
        {"name": "gemm_512x8192x4096", "op": "gemm_q8", "M": 512, "N": 8192, "K": 4096, "type": "f16", "c": False},
        # the largest product: a full prompt batch, bound by the tensor cores
        {"name": "gemm_8192x8192x8192", "op": "gemm_q8", "M": 8192, "N": 8192, "K": 8192, "type": "f16", "c": False},
        # ragged in every extent, float32 result added to a float32 C
        {"name": "gemm_1001x3001x4099_f32c", "op": "gemm_q8", "M": 1001, "N": 3001, "K": 4099, "type": "f32", "c": True},
        # one token against a large 4-bit weight matrix (an output layer)
        {"name": "gemv_1x16384x16384_g128", "op": "gemv_q4", "n_vec": 1, "rows": 16384, "cols": 16384, "group": 128,
         "x": "f16", "type": "f32", "zeros": False},
        # eight tokens that the 8-bit norm produced, small groups with zero points
        {"name": "gemv_8x4096x4096_g32_q8", "op": "gemv_q4", "n_vec": 8, "rows": 4096, "cols": 4096, "group": 32,
         "x": "e4m3", "type": "f16", "zeros": True},
        # odd extents: the last group is short, the last byte of a row half empty
        {"name": "gemv_3x3001x4099_g64", "op": "gemv_q4", "n_vec": 3, "rows": 3001, "cols": 4099, "group": 64,
         "x": "f16", "type": "f16", "zeros": True},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi):
    """Log-uniform; three in five are rounded to a multiple of 64, the others stay as drawn (odd ones among them)."""
    v = _log(rng, lo, hi)
    return max(lo, v // 64 * 64) if rng.random() < 0.6 and v >= 64 else v


def draw(rng):
    op = rng.choice(["rmsnorm_q8", "cast_q8", "gemm_q8", "gemv_q4"])
    if op in ("rmsnorm_q8", "cast_q8"):
        c = {"op": op, "rows": _log(rng, 1, 16384), "cols": _size(rng, 64, 16384), "type": rng.choice(["f16", "f16", "f32"])}
        if op == "rmsnorm_q8":
            c["residual"] = rng.random() < 0.7
        return c
    if op == "gemm_q8":
        M, N, K = _log(rng, 1, 8192), _size(rng, 64, 16384), _size(rng, 64, 16384)
        while M * N * K > 8192 ** 3:
            M = M // 2
        return {"op": op, "M": M, "N": N, "K": K, "type": rng.choice(["f16", "f16", "f32"]), "c": rng.random() < 0.3}
    return {"op": op, "n_vec": _log(rng, 1, 16), "rows": _size(rng, 64, 16384), "cols": _size(rng, 64, 16384),
            "group": rng.choice([32, 64, 128]), "x": rng.choice(["f16", "e4m3"]), "type": rng.choice(["f16", "f32"]),
            "zeros": rng.random() < 0.5}


# ------------------------------------------------------------------------------------------------ inputs
def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _pitched(rows, cols, dtype, fill=None):
    """A rows x cols view whose rows start a multiple of 128 bytes apart."""
    e = torch.empty(0, dtype=dtype).element_size()
    p = -(-cols * e // 128) * 128 // e
    buf = torch.zeros((rows, p), dtype=torch.uint8 if dtype == E4M3 else dtype, device=DEV)
    buf = buf.view(dtype) if dtype == E4M3 else buf
    v = buf[:, :cols]
    if fill is not None:
        v.copy_(fill)
    return v


def _operand8(g, rows, cols):
    """Rows of unequal magnitude as an 8-bit operand."""
    v = _normal(g, rows, cols) * torch.exp(0.5 * _normal(g, rows, 1))
    s = v.abs().amax(1) / 448
    return _pitched(rows, cols, E4M3, (v / s[:, None]).clamp(-448, 448).to(E4M3)), s


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = dict(case)
    op = case["op"]
    if op in ("rmsnorm_q8", "cast_q8"):
        rows, cols, t = case["rows"], case["cols"], TYPES[case["type"]]
        x = _normal(g, rows, cols)
        x[:, :: 97] *= 8                                        # a few channels far larger than the rest
        s["x"] = x.to(t)
        s["q"], s["scales"] = _pitched(rows, cols, E4M3), torch.empty(rows, device=DEV)
        if op == "rmsnorm_q8":
            s["weight"] = (1 + 0.2 * _normal(g, cols)).to(t)
            s["r"] = (4 * _normal(g, rows, cols)).to(t) if case["residual"] else None
            s["sum"] = torch.empty_like(s["r"]) if case["residual"] else None
    elif op == "gemm_q8":
        M, N, K, t = case["M"], case["N"], case["K"], TYPES[case["type"]]
        s["A"], s["sa"] = _operand8(g, M, K)
        s["B"], s["sb"] = _operand8(g, N, K)
        s["sb"] = s["sb"] / math.sqrt(K)
        s["C"] = _pitched(M, N, t, _normal(g, M, N).to(t)) if case["c"] else None
        s["D"] = _pitched(M, N, t)
    else:
        rows, cols, n, group = case["rows"], case["cols"], case["n_vec"], case["group"]
        groups = -(-cols // group)
        W = _pitched(rows, -(-cols // 2), torch.uint8)
        W.copy_(torch.randint(0, 256, W.shape, generator=g, device=DEV, dtype=torch.uint8))
        if cols % 2:
            W[:, -1] &= 15
        s["W"] = W
        s["ws"] = ((0.5 + torch.rand(rows, groups, generator=g, device=DEV)) / (4 * math.sqrt(cols))).half()
        s["z"] = torch.randint(5, 11, (rows, groups), generator=g, device=DEV, dtype=torch.uint8) if case["zeros"] else None
        if case["x"] == "e4m3":
            s["v"], s["vs"] = _operand8(g, n, cols)
        else:
            s["v"], s["vs"] = _normal(g, n, cols).half(), None
        s["y"] = torch.empty((n, rows), dtype=TYPES[case["type"]], device=DEV)
    return s


# ------------------------------------------------------------------------------------------------ one pass
def _to_q8(y):
    """Rows as e4m3 values and the float32 scale that takes each row's largest magnitude to 448."""
    scale = y.abs().amax(1) / 448
    q = (y / torch.where(scale == 0, 1.0, scale)[:, None]).clamp(-448, 448)
    return q.to(E4M3), scale


def _dense4(W, scales, zeros, cols, group):
    q = torch.stack((W & 15, W >> 4), dim=2).reshape(W.shape[0], -1)[:, :cols].float()
    at = torch.arange(cols, device=W.device) // group
    z = zeros.float()[:, at] if zeros is not None else 8.0
    return (q - z) * scales.float()[:, at]


def run(s):
    op = s["op"]
    if own:
        from decx_b200 import blas, gemm
        if op == "rmsnorm_q8":
            q, scales, total = blas.rmsnorm_q8(s["x"], s["weight"], residual=s["r"], eps=EPS, out=s["q"],
                                               scales=s["scales"], sum_out=s["sum"])
            return {"q": q, "scales": scales, "sum": total}
        if op == "cast_q8":
            q, scales = blas.cast_q8(s["x"], out=s["q"], scales=s["scales"])
            return {"q": q, "scales": scales}
        if op == "gemm_q8":
            one = 1.0 if s["C"] is not None else None
            return gemm.gemm_q8(s["A"], s["sa"], s["B"], s["sb"], C=s["C"], alpha=one, beta=one, out=s["D"])
        return blas.gemv_q4(s["W"], s["ws"], s["v"], s["group"], zeros=s["z"], x_scales=s["vs"], out=s["y"])
    if op == "rmsnorm_q8":
        h = s["x"].float()
        total = None
        if s["r"] is not None:
            h = h + s["r"].float()
            total = h.to(s["x"].dtype)
        y = h * torch.rsqrt(h.square().mean(1, keepdim=True) + EPS) * s["weight"].float()
        q, scales = _to_q8(y)
        return {"q": q, "scales": scales, "sum": total}
    if op == "cast_q8":
        q, scales = _to_q8(s["x"].float())
        return {"q": q, "scales": scales}
    if op == "gemm_q8":
        d = (s["A"].float() @ s["B"].float().t()) * s["sa"][:, None] * s["sb"][None, :]
        if s["C"] is not None:
            d = d + s["C"].float()
        return d.to(TYPES[s["type"]])
    x = s["v"].float()
    y = x @ _dense4(s["W"], s["ws"], s["z"], s["cols"], s["group"]).t()
    if s["vs"] is not None:
        y = y * s["vs"][:, None]
    return y.to(TYPES[s["type"]])


def work(case):
    op = case["op"]
    if op in ("rmsnorm_q8", "cast_q8"):
        n, e = case["rows"] * case["cols"], 2 if case["type"] == "f16" else 4
        if op == "cast_q8":
            return {"bytes": n * (e + 1) + 4 * case["rows"], "flops": 3 * n}
        moved = e * (3 if case["residual"] else 1) + 1
        return {"bytes": n * moved + 4 * case["rows"] + e * case["cols"], "flops": 6 * n}
    if op == "gemm_q8":
        M, N, K, e = case["M"], case["N"], case["K"], 2 if case["type"] == "f16" else 4
        return {"bytes": M * K + N * K + 4 * (M + N) + M * N * e * (2 if case["c"] else 1), "flops": 2 * M * N * K}
    rows, cols, n = case["rows"], case["cols"], case["n_vec"]
    groups = -(-cols // case["group"])
    x = n * cols * (2 if case["x"] == "f16" else 1) + (0 if case["x"] == "f16" else 4 * n)
    return {"bytes": rows * -(-cols // 2) + rows * groups * (3 if case["zeros"] else 2) + x
            + n * rows * (2 if case["type"] == "f16" else 4), "flops": 2 * n * rows * cols}


# ------------------------------------------------------------------------------------------------ the definition, in 64 bits
def _nearest_e4m3(v):
    """Nearest e4m3 value (ties to the even mantissa): steps of 2^(e - 3) from exponent -6 on, at most 448."""
    e = torch.frexp(v.abs())[1].double() - 1
    step = torch.exp2(torch.clamp(e, min=-6.0) - 3)
    return torch.clamp(torch.round(v / step) * step, -448.0, 448.0)


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op in ("rmsnorm_q8", "cast_q8"):
        h = s["x"].double()
        if op == "rmsnorm_q8":
            if s["r"] is not None:
                h += s["r"].double()
            rms = torch.sqrt((h * h).sum(1) / case["cols"] + EPS)
            v = h / rms[:, None] * s["weight"].double()
        else:
            v = h
        top = v.abs().max(1).values
        out = {"q": _nearest_e4m3(v / top[:, None] * 448), "scales": top / 448}
        if op == "rmsnorm_q8":
            out["sum"] = h if s["r"] is not None else None
        return out
    if op == "gemm_q8":
        a = s["A"].double() * s["sa"].double()[:, None]
        b = s["B"].double() * s["sb"].double()[:, None]
        d = torch.mm(a, b.t())
        return d if s["C"] is None else d + s["C"].double()
    rows, cols, group = case["rows"], case["cols"], case["group"]
    w = torch.empty((rows, 2 * s["W"].shape[1]), dtype=torch.float64, device=DEV)
    w[:, 0::2] = (s["W"] % 16).double()
    w[:, 1::2] = (s["W"] // 16).double()
    w = w[:, :cols]
    for k in range(s["ws"].shape[1]):
        part = w[:, k * group:(k + 1) * group]
        part -= s["z"][:, k:k + 1].double() if s["z"] is not None else 8.0
        part *= s["ws"][:, k:k + 1].double()
    x = s["v"].double()
    if s["vs"] is not None:
        x = x * s["vs"].double()[:, None]
    return torch.mm(x, w.t())
