"""Measured cases of the MXFP8 layer operators: RMS norm with 8-bit output and
its gradient, the block-scaled matrix product with bias, activation and
residual in its epilogue, and 8-bit activation checkpoints with their use in
the backward pass.

``run`` computes a case in its plain form (elementary torch operations in 32
bits, rounded once) where ``own`` is false, and through the package's
operators where it is true.  Operands are quantised block-scaled matrices as
a program holds them between calls: uint8 codes and uint8 scales in the
tensor-core chunk layout.  8-bit outputs are returned as tensors of their
element types (e4m3 values, power-of-two e8m0 scales).
"""
from __future__ import annotations

import math

import torch

own = False

E4M3 = torch.float8_e4m3fn
E8M0 = torch.float8_e8m0fnu
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
LAYOUTS = {"linear": 0, "mma": 1, "kmajor": 2}
FORMATS = {"mxfp8": (1.0, 32), "nvfp4": (0.5, 16), "mxfp4": (0.5, 32)}  # bytes per value, block
EPS = 1e-5


# ------------------------------------------------------------------ cases
def listed():
    return [
        # One token of a decode step entering a layer of width 8192.
        {"name": "norm_token", "op": "norm", "rows": 1, "k": 8192, "dtype": "bf16",
         "residual": True, "layout": "mma", "pad": 0},
        # A training step's 16384 tokens of that width.
        {"name": "norm_train", "op": "norm", "rows": 16384, "k": 8192, "dtype": "bf16",
         "residual": True, "layout": "mma", "pad": 0},
        # fp32 master activations, a short odd batch cut out of a wider buffer.
        {"name": "norm_bwd_ragged", "op": "norm_bwd", "rows": 333, "k": 5152, "dtype": "f32",
         "dres": False, "pad": 32},
        # The gradient of norm_train, joined with the residual branch's.
        {"name": "norm_bwd_train", "op": "norm_bwd", "rows": 16384, "k": 8192, "dtype": "bf16",
         "dres": True, "pad": 0},
        # One token through a gated up-projection (2 x 14336 from 4096), output
        # quantised for the next product: weight-streaming latency.
        {"name": "gemm_token_gated", "op": "gemm", "fmt": "mxfp8", "m": 1, "n": 28672, "k": 4096,
         "act": "swiglu", "bias": False, "residual": False, "dtype": "bf16", "out": "mxfp8",
         "ckpt": False},
        # 64 decoding sequences through the down-projection with the residual added.
        {"name": "gemm_decode_down", "op": "gemm", "fmt": "mxfp8", "m": 64, "n": 4096, "k": 14336,
         "act": "none", "bias": False, "residual": True, "dtype": "bf16", "out": "bf16",
         "ckpt": False},
        # 4-bit weights and activations, every size odd against the tiles.
        {"name": "gemm_ragged_nvfp4", "op": "gemm", "fmt": "nvfp4", "m": 1000, "n": 4136,
         "k": 2080, "act": "gelu", "bias": True, "residual": True, "dtype": "bf16",
         "out": "bf16", "ckpt": False},
        # A training step's gated up-projection: 8-bit output for the next
        # product and the 8-bit checkpoint of the pre-activation.
        {"name": "gemm_train_gated", "op": "gemm", "fmt": "mxfp8", "m": 4096, "n": 28672,
         "k": 4096, "act": "swiglu", "bias": False, "residual": False, "dtype": "bf16",
         "out": "mxfp8", "ckpt": True},
        # Backward of a biased GELU layer over an odd number of tokens, fp32 gradients.
        {"name": "act_bwd_ragged", "op": "act_bwd", "m": 333, "n": 4128, "act": "gelu",
         "dtype": "f32"},
        # Backward of gemm_train_gated from its checkpoint: the gradient
        # quantised along both axes for the two products that follow.
        {"name": "act_bwd_train", "op": "act_bwd", "m": 4096, "n": 28672, "act": "swiglu",
         "dtype": "bf16"},
        # An 8-bit input kept from the forward pass, turned for the weight
        # gradient: an odd batch, and a training step's.
        {"name": "transpose_ragged", "op": "transpose", "rows": 1000, "k": 4128},
        {"name": "transpose_train", "op": "transpose", "rows": 16384, "k": 8192},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm_bwd", "gemm", "gemm", "act_bwd", "transpose"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op in ("norm", "norm_bwd"):
        k = 32 * _log(rng, 1, 512)
        rows = _log(rng, 1, min(32768, (1 << 27) // k))
        c = {"op": op, "rows": rows, "k": k, "dtype": dtype,
             "pad": rng.choice([0, 0, 32 * rng.randint(1, 8)])}
        if op == "norm":
            c["residual"] = rng.random() < 0.7
            c["layout"] = rng.choice(["mma", "mma", "kmajor", "linear"])
        else:
            c["dres"] = rng.random() < 0.7
        return c
    if op == "transpose":
        k = 32 * _log(rng, 1, 896)
        return {"op": op, "rows": _log(rng, 1, min(32768, (1 << 27) // k)), "k": k}
    act = rng.choice(["none", "relu", "silu", "gelu", "swiglu", "swiglu"])
    if op == "act_bwd":
        n = 256 * _log(rng, 1, 112) if act == "swiglu" else 32 * _log(rng, 1, 896)
        return {"op": op, "m": _log(rng, 1, min(32768, (1 << 27) // n)), "n": n, "act": act,
                "dtype": dtype}
    out = rng.choice(["bf16", "bf16", "f32", "mxfp8"])
    ckpt = rng.random() < 0.4
    k = 32 * _log(rng, 1, 448)
    if act == "swiglu":
        n = 256 * _log(rng, 1, 112)
    elif out == "mxfp8" or ckpt:
        n = 32 * _log(rng, 1, 896)
    else:
        n = _log(rng, 8, 28672)
    m = _log(rng, 1, max(1, min(8192, (1 << 38) // (n * k))))
    return {"op": op, "fmt": rng.choice(["mxfp8", "mxfp8", "nvfp4", "mxfp4"]), "m": m, "n": n,
            "k": k, "act": act, "bias": rng.random() < 0.5, "residual": rng.random() < 0.5,
            "dtype": dtype, "out": out, "ckpt": ckpt}


def work(case):
    op = case["op"]
    e = 2 if case.get("dtype") == "bf16" else 4
    if op == "norm":
        n, k, rows = case["rows"] * case["k"], case["k"], case["rows"]
        # x (and the residual in, the sum out), the weight, values, scales, rstd.
        moved = n * (e * (3 if case["residual"] else 1) + 33 / 32) + k * e + 4 * rows
        return {"bytes": moved, "flops": 5 * n}
    if op == "norm_bwd":
        n, k, rows = case["rows"] * case["k"], case["k"], case["rows"]
        return {"bytes": n * e * (4 if case["dres"] else 3) + k * (e + 4) + 4 * rows,
                "flops": 9 * n}
    if op == "transpose":
        rows, k = case["rows"], case["k"]
        return {"bytes": 33 / 32 * k * (rows + _up32(rows)), "flops": 2 * rows * k}
    m, n, act = case["m"], case["n"], case["act"]
    n_out = n // 2 if act == "swiglu" else n
    if op == "act_bwd":
        moved = m * n_out * e + 33 / 32 * n * (2 * m + _up32(m)) + 4 * n
        return {"bytes": moved, "flops": 12 * m * n}
    k = case["k"]
    vb, sv = FORMATS[case["fmt"]]
    moved = (m + n) * k * (vb + 1 / sv)
    moved += m * n_out * {"bf16": 2, "f32": 4, "mxfp8": 33 / 32}[case["out"]]
    moved += m * n * 33 / 32 if case["ckpt"] else 0
    moved += m * n_out * e if case["residual"] else 0
    moved += n * e if case["bias"] else 0
    return {"bytes": moved, "flops": 2 * m * n * k}


def _up32(x):
    return (x + 31) // 32 * 32


# ------------------------------------------------------------------ formats
def _to_chunks(codes, layout):
    """Scale codes [rows][blocks] in the named layout's byte order: linear, or
    chunks of 128 rows x 4 blocks (row r of a chunk at byte 16 (r % 32) +
    4 (r / 32)), row blocks inner (mma) or outer (kmajor)."""
    if layout == "linear":
        return codes.reshape(-1)
    rows, blocks = codes.shape
    rb, cb = (rows + 127) // 128, (blocks + 3) // 4
    full = codes.new_zeros(rb * 128, cb * 4)
    full[:rows, :blocks] = codes
    chunk = full.view(rb, 4, 32, cb, 4)
    order = (3, 0, 2, 1, 4) if layout == "mma" else (0, 3, 2, 1, 4)
    return chunk.permute(order).reshape(-1)


def _from_chunks(flat, rows, blocks):
    """Inverse of _to_chunks for the mma layout."""
    rb, cb = (rows + 127) // 128, (blocks + 3) // 4
    full = flat.view(cb, rb, 32, 4, 4).permute(1, 3, 2, 0, 4).reshape(rb * 128, cb * 4)
    return full[:rows, :blocks]


def _mx_blocks(y):
    """Exponents [rows][k / 32] of the MXFP8 rule: floor(log2 of the block's
    largest magnitude) - 8, -127 for a block of zeros; and the blocks."""
    b = y.reshape(y.shape[0], -1, 32)
    amax = b.abs().amax(-1)
    e = torch.where(amax > 0, torch.frexp(amax)[1] - 9, torch.full_like(amax, -127).int())
    return e.clamp(-127, 127), b


def _mxfp8(y, layout="mma"):
    """(e4m3 values [rows][k], e8m0 scales in `layout`) of a 32-bit matrix."""
    e, b = _mx_blocks(y)
    q = (b * torch.exp2(-e.float()).unsqueeze(-1)).clamp(-448, 448).to(E4M3)
    codes = (e + 127).to(torch.uint8)
    return q.reshape(y.shape), _to_chunks(codes, layout).view(E8M0)


def _mxfp8_value(q, sf, rows, k, dtype=torch.float32):
    s = torch.exp2(_from_chunks(sf, rows, k // 32).to(dtype) - 127)
    return (q.view(E4M3).view(rows, k // 32, 32).to(dtype) * s.unsqueeze(-1)).view(rows, k)


def _value(x, fmt, rows, k, dtype=torch.float32):
    """The matrix that an operand's codes, scales and tensor scale stand for."""
    q, sf, ts = x
    if fmt == "mxfp8":
        return _mxfp8_value(q, sf, rows, k, dtype)
    table = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, 0, -.5, -1, -1.5, -2, -3, -4, -6],
                         dtype=dtype, device=q.device)
    pairs = q.view(rows, k // 2)
    v = table[torch.stack([pairs & 15, pairs >> 4], -1).long()].view(rows, k)
    sv = FORMATS[fmt][1]
    codes = _from_chunks(sf, rows, k // sv)
    s = codes.contiguous().view(E4M3).to(dtype) if fmt == "nvfp4" else torch.exp2(
        codes.to(dtype) - 127)
    v = (v.view(rows, k // sv, sv) * s.unsqueeze(-1)).view(rows, k)
    return v * ts.to(dtype) if fmt == "nvfp4" else v


# ------------------------------------------------------------------ inputs
def _normal(g, *shape, std=1.0, outliers=False, dtype=torch.float32):
    x = torch.randn(*shape, generator=g, device="cuda") * std
    if outliers:  # activations: one value in a thousand 50 times the others
        x *= 1 + 49 * (torch.rand(*shape, generator=g, device="cuda") < 0.001)
    return x.to(dtype)


def _padded(g, rows, k, pad, dtype, **kw):
    return _normal(g, rows, k + pad, dtype=dtype, **kw)[:, :k]


def _operand(x, fmt):
    """Codes, scales (mma layout) and tensor scale of a matrix in a format."""
    rows, k = x.shape
    if fmt == "mxfp8":
        q, sf = _mxfp8(x)
        return q.view(torch.uint8), sf.view(torch.uint8), None
    sv = FORMATS[fmt][1]
    b = x.view(rows, k // sv, sv)
    amax = b.abs().amax(-1)
    if fmt == "nvfp4":
        ts = (amax.max() / 2688).reshape(1)
        s = (amax / (6 * ts)).clamp(max=448).to(E4M3)
        mul, codes = s.float() * ts, s.view(torch.uint8)
    else:
        ts = None
        e = torch.frexp(amax)[1] - 3
        mul, codes = torch.exp2(e.float()), (e + 127).to(torch.uint8)
    a = (b / mul.unsqueeze(-1)).abs()
    code = (a > 0.25).to(torch.uint8)
    for edge in (0.75, 1.25, 1.75, 2.5, 3.5, 5.0):
        code += a >= edge
    code += 8 * (b < 0)
    code = code.view(rows, k // 2, 2)
    return (code[..., 0] | code[..., 1] << 4).reshape(-1), _to_chunks(codes, "mma"), ts


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, s = case["op"], dict(case)
    dt = DTYPES[case.get("dtype", "f32")]
    if op in ("norm", "norm_bwd"):
        rows, k, pad = case["rows"], case["k"], case["pad"]
        s["w"] = (1 + 0.2 * torch.randn(k, generator=g, device="cuda")).to(dt)
        if op == "norm":
            s["x"] = _padded(g, rows, k, pad, dt, outliers=True)
            s["r"] = _padded(g, rows, k, pad, dt, std=2.0) if case["residual"] else None
        else:
            s["h"] = _padded(g, rows, k, pad, dt, std=2.0, outliers=True)
            s["rstd"] = (s["h"].float().square().mean(-1) + EPS).rsqrt()
            s["dy"] = _padded(g, rows, k, pad, dt, std=0.01)
            s["dres"] = _padded(g, rows, k, pad, dt, std=0.01) if case["dres"] else None
    elif op == "gemm":
        m, n, k, fmt = case["m"], case["n"], case["k"], case["fmt"]
        n_out = n // 2 if case["act"] == "swiglu" else n
        s["a"] = _operand(_normal(g, m, k), fmt)
        s["b"] = _operand(_normal(g, n, k, std=1.5 / math.sqrt(k)), fmt)
        s["bias_t"] = _normal(g, n, std=0.5, dtype=dt) if case["bias"] else None
        s["res_t"] = _normal(g, m, n_out, std=2.0, dtype=dt) if case["residual"] else None
    elif op == "act_bwd":
        m, n = case["m"], case["n"]
        s["z"] = _operand(_normal(g, m, n, std=1.5), "mxfp8")
        s["dout"] = _normal(g, m, n // 2 if case["act"] == "swiglu" else n, std=0.01, dtype=dt)
    else:
        s["a"] = _operand(_normal(g, case["rows"], case["k"], outliers=True), "mxfp8")
    return s


# ------------------------------------------------------------------ operators
def run(s):
    if own:
        return _run_own(s)
    return {"norm": _norm, "norm_bwd": _norm_bwd, "gemm": _gemm, "act_bwd": _act_bwd,
            "transpose": _transpose}[s["op"]](s)


def _run_own(s):
    from cuda_optimazation_b200 import Mxfp4Result, Mxfp8Result, Nvfp4Result, fused
    op = s["op"]

    def held(x, rows, k, fmt="mxfp8"):
        if fmt == "nvfp4":
            return Nvfp4Result(x[0], x[1], x[2], rows, k, 1)
        return (Mxfp8Result if fmt == "mxfp8" else Mxfp4Result)(x[0], x[1], rows, k, 1)

    def q(r):
        return r.quantized.view(E4M3).view(r.rows, r.k)

    if op == "norm":
        o = fused.rmsnorm_mxfp8(s["x"], s["w"], residual=s["r"], eps=EPS,
                                layout=LAYOUTS[s["layout"]])
        out = {"q": q(o.y), "scales": o.y.block_scales.view(E8M0), "rstd": o.rstd}
        if s["r"] is not None:
            out["h"] = o.h
        return out
    if op == "norm_bwd":
        dx, dw = fused.rmsnorm_backward(s["dy"], s["h"], s["rstd"], s["w"], dres=s["dres"])
        return {"dx": dx, "dw": dw}
    if op == "transpose":
        t = fused.transpose_mxfp8(held(s["a"], s["rows"], s["k"]))
        return {"q": q(t), "scales": t.block_scales.view(E8M0)}
    if op == "act_bwd":
        o = fused.act_backward(s["dout"], held(s["z"], s["m"], s["n"]), s["act"])
        return {"dz": q(o.dz), "dz_scales": o.dz.block_scales.view(E8M0), "dzt": q(o.dz_t),
                "dzt_scales": o.dz_t.block_scales.view(E8M0), "dbias": o.dbias}
    o = fused.gemm_fused(held(s["a"], s["m"], s["k"], s["fmt"]),
                         held(s["b"], s["n"], s["k"], s["fmt"]), bias=s["bias_t"], act=s["act"],
                         residual=s["res_t"], out=s["out"], checkpoint=s["ckpt"])
    out = {"out": q(o.out), "scales": o.out.block_scales.view(E8M0)} if s["out"] == "mxfp8" else {
        "out": o.out}
    if s["ckpt"]:
        out |= {"z": q(o.checkpoint), "z_scales": o.checkpoint.block_scales.view(E8M0)}
    return out


def _norm(s):
    h = s["x"].float()
    if s["r"] is not None:
        h = h + s["r"].float()
    rstd = (h.square().mean(-1) + EPS).rsqrt()
    q, sf = _mxfp8(h * rstd.unsqueeze(-1) * s["w"].float(), s["layout"])
    out = {"q": q, "scales": sf, "rstd": rstd}
    if s["r"] is not None:
        out["h"] = h.to(s["x"].dtype)
    return out


def _norm_bwd(s):
    xhat = s["h"].float() * s["rstd"].unsqueeze(-1)
    dy = s["dy"].float()
    gw = dy * s["w"].float()
    dx = s["rstd"].unsqueeze(-1) * (gw - xhat * (gw * xhat).mean(-1, keepdim=True))
    if s["dres"] is not None:
        dx = dx + s["dres"].float()
    return {"dx": dx.to(s["h"].dtype), "dw": (dy * xhat).sum(0)}


def _act(z, act):
    if act == "none":
        return z
    if act == "relu":
        return z.clamp(min=0)
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        # z / 2 (1 + tanh(v / 2)), without the difference's loss of digits at z < 0.
        return z / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    g, u = z.view(z.shape[0], -1, 2, 128).unbind(2)  # 128 gate columns, their 128 factors
    return (g / (1 + torch.exp(-g)) * u).reshape(z.shape[0], -1)


def _act_grad(d, z, act):
    if act == "none":
        return d
    if act == "relu":
        return d * (z > 0)
    if act == "silu":
        sg = 1 / (1 + torch.exp(-z))
        return d * sg * (1 + z * (1 - sg))
    if act == "gelu":
        c = 2 * math.sqrt(2 / math.pi)
        sg = 1 / (1 + torch.exp(-c * (z + 0.044715 * z ** 3)))
        return d * sg * (1 + z * (1 - sg) * c * (1 + 3 * 0.044715 * z * z))
    g, u = z.view(z.shape[0], -1, 2, 128).unbind(2)
    d = d.view(g.shape)
    sg = 1 / (1 + torch.exp(-g))
    return torch.stack([d * u * sg * (1 + g * (1 - sg)), d * g * sg], 2).reshape(z.shape)


def _gemm(s):
    m, n, k, fmt = s["m"], s["n"], s["k"], s["fmt"]
    z = _value(s["a"], fmt, m, k) @ _value(s["b"], fmt, n, k).t()
    if s["bias_t"] is not None:
        z = z + s["bias_t"].float()
    y = _act(z, s["act"])
    if s["res_t"] is not None:
        y = y + s["res_t"].float()
    if s["out"] == "mxfp8":
        q, sf = _mxfp8(y)
        out = {"out": q, "scales": sf}
    else:
        out = {"out": y.to(DTYPES[s["out"]])}
    if s["ckpt"]:
        q, sf = _mxfp8(z)
        out |= {"z": q, "z_scales": sf}
    return out


def _turned(y):
    """A matrix's transpose with its columns filled up with zeros to a multiple of 32."""
    t = y.new_zeros(y.shape[1], _up32(y.shape[0]))
    t[:, :y.shape[0]] = y.t()
    return t


def _act_bwd(s):
    m, n = s["m"], s["n"]
    dz = _act_grad(s["dout"].float(), _mxfp8_value(s["z"][0], s["z"][1], m, n), s["act"])
    q, sf = _mxfp8(dz)
    qt, sft = _mxfp8(_turned(dz))
    return {"dz": q, "dz_scales": sf, "dzt": qt, "dzt_scales": sft, "dbias": dz.sum(0)}


def _transpose(s):
    q, sf = _mxfp8(_turned(_mxfp8_value(s["a"][0], s["a"][1], s["rows"], s["k"])))
    return {"q": q, "scales": sf}


# ------------------------------------------------------------------ 64 bits
def _codes64(y):
    """What an MXFP8 matrix's elements approximate: y in units of its exact
    block scale.  The scales themselves are choices of a power of two and
    have no rounding error of their own: they are held by the elements."""
    peak = y.reshape(y.shape[0], -1, 32).abs().amax(-1)
    unit = torch.where(peak > 0, torch.exp2(torch.floor(torch.log2(peak)) - 8),
                       torch.full_like(peak, 2.0 ** -127))
    return y / unit.repeat_interleave(32, 1)


def exact(case, seed):
    s, d64 = prepare(case, seed), torch.float64
    op = case["op"]
    if op == "norm":
        h = s["x"].to(d64) + (0 if s["r"] is None else s["r"].to(d64))
        r = 1 / torch.sqrt((h * h).sum(-1) / case["k"] + EPS)
        out = {"q": _codes64(h * r[:, None] * s["w"].to(d64)), "scales": None, "rstd": r}
        if s["r"] is not None:
            out["h"] = h
        return out
    if op == "norm_bwd":
        h, dy, w, r = (s[i].to(d64) for i in ("h", "dy", "w", "rstd"))
        r = r[:, None]
        dot = (dy * w * h).sum(-1, keepdim=True) / case["k"]
        dx = r * dy * w - r ** 3 * h * dot
        if s["dres"] is not None:
            dx += s["dres"].to(d64)
        return {"dx": dx, "dw": (dy * h * r).sum(0)}
    if op == "transpose":
        x = _mxfp8_value(s["a"][0], s["a"][1], case["rows"], case["k"], d64)
        return {"q": _codes64(_turned(x)), "scales": None}
    act = case["act"]
    if op == "act_bwd":
        z = _mxfp8_value(s["z"][0], s["z"][1], case["m"], case["n"], d64)
        d = s["dout"].to(d64)
        if act == "none":
            dz = d
        elif act == "relu":
            dz = torch.where(z > 0, d, torch.zeros_like(d))
        elif act == "gelu":
            a = math.sqrt(2 / math.pi)
            t = torch.tanh(a * (z + 0.044715 * z ** 3))
            dz = d * (0.5 + 0.5 * t + 0.5 * a * z * (1 + 0.134145 * z * z) * (1 - t * t))
        else:
            def slope(v):
                p = torch.sigmoid(v)
                return p + v * p * (1 - p)
            if act == "silu":
                dz = d * slope(z)
            else:
                dz = torch.empty_like(z)
                zc, dc = z.view(len(z), -1, 256), d.view(len(d), -1, 128)
                to = dz.view(len(z), -1, 256)
                to[..., :128] = dc * zc[..., 128:] * slope(zc[..., :128])
                to[..., 128:] = dc * zc[..., :128] * torch.sigmoid(zc[..., :128])
        return {"dz": _codes64(dz), "dz_scales": None, "dzt": _codes64(_turned(dz)),
                "dzt_scales": None, "dbias": dz.sum(0)}
    m, n, k, fmt = case["m"], case["n"], case["k"], case["fmt"]
    z = _value(s["a"], fmt, m, k, d64) @ _value(s["b"], fmt, n, k, d64).t()
    if s["bias_t"] is not None:
        z += s["bias_t"].to(d64)
    if act == "none":
        y = z
    elif act == "relu":
        y = torch.where(z > 0, z, torch.zeros_like(z))
    elif act == "silu":
        y = z * torch.sigmoid(z)
    elif act == "gelu":
        y = 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    else:
        zc = z.view(m, -1, 256)
        y = (zc[..., :128] * torch.sigmoid(zc[..., :128]) * zc[..., 128:]).reshape(m, -1)
    if s["res_t"] is not None:
        y = y + s["res_t"].to(d64)
    out = {"out": _codes64(y), "scales": None} if case["out"] == "mxfp8" else {"out": y}
    if case["ckpt"]:
        out |= {"z": _codes64(z), "z_scales": None}
    return out
