"""64-bit references of the layer operators and the check of an MXFP8 matrix
against them."""
from __future__ import annotations

import math

import torch

F64 = torch.float64
E4M3 = torch.float8_e4m3fn


def chunk_order(rows: int, blocks: int, layout: int):
    """(row, block) -> byte offset of a scale, and the buffer's size."""
    r = torch.arange(rows).view(-1, 1)
    c = torch.arange(blocks).view(1, -1)
    if layout == 0:
        return r * blocks + c, rows * blocks
    rb, cb = (rows + 127) // 128, (blocks + 3) // 4
    chunk = (c // 4) * rb + r // 128 if layout == 1 else (r // 128) * cb + c // 4
    return chunk * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + c % 4, rb * cb * 512


def exponents(amax: torch.Tensor) -> torch.Tensor:
    """floor(log2 amax) - 8, at least -127 (zero blocks too), in 64 bits."""
    e = torch.frexp(amax.to(F64))[1] - 1 - 8
    return torch.where(amax > 0, e, torch.full_like(e, -127)).clamp(min=-127)


def quantise(x: torch.Tensor, layout: int = 1):
    """MXFP8 codes [rows, k] and the scale buffer of a matrix."""
    rows, k = x.shape
    b = x.to(F64).view(rows, k // 32, 32)
    e = exponents(b.abs().amax(-1))
    q = (b * torch.exp2(-e.to(F64)).unsqueeze(-1)).clamp(-448, 448).float().to(E4M3)
    at, size = chunk_order(rows, k // 32, layout)
    sf = torch.zeros(size, dtype=torch.uint8, device=x.device)
    sf[at.to(x.device)] = (e + 127).to(torch.uint8)
    return q.view(torch.uint8).view(rows, k), sf


def parts(r):
    """(element values, exponents) of an Mxfp8Result, both 64-bit / integer."""
    at, size = chunk_order(r.rows, r.k // 32, r.layout)
    assert r.block_scales.numel() == size
    used = torch.zeros(size, dtype=torch.bool, device=r.block_scales.device)
    used[at.to(used.device)] = True
    assert int(r.block_scales[~used].sum()) == 0, "scale padding is not zero"
    e = r.block_scales[at.to(used.device)].int() - 127
    return r.quantized.view(E4M3).view(r.rows, r.k).to(F64), e


def value(r) -> torch.Tensor:
    q, e = parts(r)
    return (q.view(r.rows, -1, 32) * torch.exp2(e.to(F64)).unsqueeze(-1)).view(r.rows, r.k)


def check_mx(r, ref: torch.Tensor, tol: torch.Tensor) -> None:
    """r quantises some y with |y - ref| <= tol: every scale is that of a block
    peak within the tolerance, and every value is y rounded to 3 mantissa bits
    (half a step: 2^-4 of it), to the grid of subnormals (half a step: 2^-10 of
    the scale) or, above 448 scales, to 448."""
    q, e = parts(r)
    b, t = ref.view(r.rows, -1, 32), tol.view(r.rows, -1, 32)
    lo = exponents((b.abs() - t).clamp(min=0).amax(-1))
    hi = exponents((b.abs() + t).amax(-1))
    assert bool(((e >= lo) & (e <= hi)).all()), "a block scale is off"
    s = torch.exp2(e.to(F64)).unsqueeze(-1)
    err = (q.view_as(b) * s - b).abs()
    top = (b.abs() + t - 448 * s).clamp(min=0)
    most = t + (b.abs() + t) * 2.0 ** -4 + s * 2.0 ** -10 + top
    assert bool((err <= most).all()), f"worst excess {float((err - most).max()):.3e}"


def act(z: torch.Tensor, name: str) -> torch.Tensor:
    if name == "none":
        return z
    if name == "relu":
        return torch.relu(z)  # slope 0 at 0 (clamp's would be 1)
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    g, u = z.view(z.shape[0], -1, 2, 128).unbind(2)
    return (g * torch.sigmoid(g) * u).reshape(z.shape[0], -1)


def act_tol(z: torch.Tensor, tol: torch.Tensor, name: str) -> torch.Tensor:
    """Bound on |act(z') - act(z)| for |z' - z| <= tol, with the fp32 evaluation's
    own error: slopes of relu, silu and gelu are below 1.2, and exp and the
    quotient are good to 2^-20 of the result for the arguments tested."""
    if name != "swiglu":
        return 1.2 * tol + 2.0 ** -20 * z.abs()
    g, u = z.view(z.shape[0], -1, 2, 128).unbind(2)
    tg, tu = tol.view(z.shape[0], -1, 2, 128).unbind(2)
    return (1.2 * tg * (u.abs() + tu) + (g.abs() + tg) * tu +
            2.0 ** -20 * (g * u).abs()).reshape(z.shape[0], -1)


def norm(x, residual, w, eps):
    h = x.to(F64) + (0 if residual is None else residual.to(F64))
    rstd = 1 / torch.sqrt((h * h).mean(-1) + eps)
    return h, rstd, h * rstd[:, None] * w.to(F64)
