"""Layer operators around the block-scaled GEMM, over the C ABI in
include/qgemm.h: what a transformer layer computes next to its products,
writing and reading the operands that the products use.

``rmsnorm_mxfp8`` (RMS norm, residual addition, 8-bit output) and
``rmsnorm_backward``; ``gemm_fused`` (bias, activation, residual in the GEMM's
epilogue, 8-bit output, 8-bit checkpoint of the pre-activation);
``act_backward`` and ``transpose_mxfp8`` (the checkpoint and the kept 8-bit
input in the backward pass).  ``mlp.py`` runs them together.

Every wrapper allocates its outputs on the stream that it launches on
(``stream``, by default the current one).
"""
from __future__ import annotations

import contextlib
import ctypes
from dataclasses import dataclass
from typing import Optional, Union

import torch

from .qgemm import (
    ACT_GELU, ACT_NONE, ACT_RELU, ACT_SILU, ACT_SWIGLU, DTYPE_BF16, DTYPE_F32, DTYPE_MXFP8,
    FORMAT_MXFP4, FORMAT_MXFP8, FORMAT_NVFP4, LAYOUT_MMA, LAYOUT_REF_LINEAR, Epilogue, Mxfp4Result,
    Mxfp8Result, Nvfp4Result, _check, lib,
)

try:  # the stream's handle without a Stream object (3.5 us a call)
    from torch._C import _cuda_getCurrentRawStream as _raw_stream
except ImportError:
    def _raw_stream(index: int) -> int:
        return torch.cuda.current_stream(index).cuda_stream

ACTIVATIONS = {"none": ACT_NONE, "relu": ACT_RELU, "silu": ACT_SILU, "gelu": ACT_GELU,
               "swiglu": ACT_SWIGLU}
GATE_COLUMNS = 128  # columns of a gate block of the gated activation
_OUTPUTS = {"f32": DTYPE_F32, "bf16": DTYPE_BF16, "mxfp8": DTYPE_MXFP8}
_TORCH = {"f32": torch.float32, "bf16": torch.bfloat16}
_CODES = {torch.float32: DTYPE_F32, torch.bfloat16: DTYPE_BF16}
_HERE = contextlib.nullcontext()

Operand = Union[Mxfp8Result, Nvfp4Result, Mxfp4Result]


def _scope(device: torch.device, stream: Optional[torch.cuda.Stream]):
    """Context in which `stream` (or the device's current one) is current."""
    if stream is not None:
        if stream.device != device:
            raise ValueError("stream and tensors are on different devices")
        return torch.cuda.stream(stream)
    return _HERE if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _code(t: torch.Tensor, what: str) -> int:
    c = _CODES.get(t.dtype)
    if c is None:
        raise TypeError(f"{what}: unsupported dtype {t.dtype}; use float32 or bfloat16")
    return c


def _matrix(t: torch.Tensor, what: str, rows: int, cols: int, device, dtype=None) -> int:
    """Checks a matrix and returns its row stride."""
    if t.shape != (rows, cols):
        raise ValueError(f"{what} must be {rows} x {cols}, got {tuple(t.shape)}")
    ld, step = t.stride()
    if t.device != device or (step != 1 and cols > 1):
        raise ValueError(f"{what} must be on {device} with unit column stride")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{what} must be {dtype}, got {t.dtype}")
    return ld if rows > 1 else cols  # the stride of a single row is arbitrary in torch


def _vector(t: torch.Tensor, what: str, n: int, device) -> None:
    if t.shape != (n,) or t.device != device or (n > 1 and t.stride(0) != 1):
        raise ValueError(f"{what} must be a contiguous vector of {n} values on {device}")


def _sf_bytes(rows: int, k: int, layout: int) -> int:
    if layout == LAYOUT_REF_LINEAR:
        return rows * (k // 32)
    return ((rows + 127) // 128) * ((k // 32 + 3) // 4) * 512


def _new_mxfp8(rows: int, k: int, layout: int, device) -> Mxfp8Result:
    return Mxfp8Result(torch.empty(rows * k, dtype=torch.uint8, device=device),
                       torch.empty(_sf_bytes(rows, k, layout), dtype=torch.uint8, device=device),
                       rows, k, layout)


def _held(a: Operand, what: str) -> torch.device:
    """Checks a quantised operand's buffers against its shape; their device."""
    q, sf, rows, k = a.quantized, a.block_scales, a.rows, a.k
    kind = type(a)
    sv = 16 if kind is Nvfp4Result else 32
    if a.layout == LAYOUT_REF_LINEAR:
        scales = rows * (k // sv)
    else:
        scales = ((rows + 127) // 128) * ((k // sv + 3) // 4) * 512
    if q.numel() < (rows * k if kind is Mxfp8Result else rows * k // 2) or sf.numel() < scales:
        raise ValueError(f"{what}: buffers are smaller than the shape {rows} x {k} needs")
    if not (q.is_contiguous() and sf.is_contiguous()):
        raise ValueError(f"{what}: buffers must be contiguous")
    dev = q.device
    if dev.type != "cuda" or sf.device != dev:
        raise ValueError(f"{what}: buffers must be on one CUDA device")
    return dev


def _mxfp8(a, what: str) -> torch.device:
    if not isinstance(a, Mxfp8Result):
        raise TypeError(f"{what} must be an Mxfp8Result")
    return _held(a, what)


# ------------------------------------------------------------------ RMS norm
@dataclass
class RmsNormResult:
    y: Mxfp8Result               # the normalised rows, quantised
    h: torch.Tensor              # x + residual (x itself without one)
    rstd: torch.Tensor           # float32 [rows], for the gradient


def rmsnorm_mxfp8(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None,
                  eps: float = 1e-5, layout: int = LAYOUT_MMA,
                  h: Optional[torch.Tensor] = None,
                  stream: Optional[torch.cuda.Stream] = None) -> RmsNormResult:
    """h = x + residual, y = MXFP8(h / sqrt(mean(h^2) + eps) * weight), in one
    pass (qg_rmsnorm_mxfp8).  x: fp32/bf16 [rows, k], any row stride of whole
    16-byte vectors; residual as x; weight fp32/bf16 [k].  ``h`` may be given
    as the buffer for the sum (x or residual itself, to update in place)."""
    if x.dim() != 2 or not x.is_cuda:
        raise ValueError("x must be a 2-D CUDA tensor")
    rows, k = x.shape
    dev = x.device
    code = _code(x, "x")
    ldx = _matrix(x, "x", rows, k, dev)
    _vector(weight, "weight", k, dev)
    rp = hp = None
    ldr = ldh = 0
    if residual is not None:
        ldr, rp = _matrix(residual, "residual", rows, k, dev, x.dtype), residual.data_ptr()
    if h is not None:
        ldh = _matrix(h, "h", rows, k, dev, x.dtype)
    with _scope(dev, stream):
        y = _new_mxfp8(rows, k, layout, dev)
        rstd = torch.empty(rows, dtype=torch.float32, device=dev)
        if h is None and residual is not None:
            h, ldh = torch.empty(rows, k, dtype=x.dtype, device=dev), k
        if h is not None:
            hp = h.data_ptr()
        rc = lib().qg_rmsnorm_mxfp8(
            x.data_ptr(), code, ldx, rp, ldr, weight.data_ptr(), _code(weight, "weight"), eps,
            rows, k, layout, y.quantized.data_ptr(), y.block_scales.data_ptr(), hp, ldh,
            rstd.data_ptr(), _raw_stream(dev.index))
    _check(rc, "qg_rmsnorm_mxfp8")
    return RmsNormResult(y, x if h is None else h, rstd)


def rmsnorm_backward(dy: torch.Tensor, h: torch.Tensor, rstd: torch.Tensor, weight: torch.Tensor,
                     dres: Optional[torch.Tensor] = None, want_dweight: bool = True,
                     stream: Optional[torch.cuda.Stream] = None
                     ) -> tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Gradient of ``rmsnorm_mxfp8`` (the quantisation passed straight through):
    (dx, dweight) from dy = dL/dy, the saved h and rstd, and optionally dres,
    the gradient that reaches h past the norm.  dx (h's dtype) is the gradient
    of x and of the residual; dweight is fp32 (None if not wanted)."""
    if h.dim() != 2 or not h.is_cuda:
        raise ValueError("h must be a 2-D CUDA tensor")
    rows, k = h.shape
    dev = h.device
    code = _code(h, "h")
    ldh = _matrix(h, "h", rows, k, dev)
    lddy = _matrix(dy, "dy", rows, k, dev, h.dtype)
    _vector(rstd, "rstd", rows, dev)
    _vector(weight, "weight", k, dev)
    if rstd.dtype != torch.float32:
        raise TypeError("rstd must be float32")
    rp, ldr = None, 0
    if dres is not None:
        ldr, rp = _matrix(dres, "dres", rows, k, dev, h.dtype), dres.data_ptr()
    with _scope(dev, stream):
        dx = torch.empty(rows, k, dtype=h.dtype, device=dev)
        dw = dwp = wsp = None
        need = 0
        if want_dweight:
            dw = torch.empty(k, dtype=torch.float32, device=dev)
            dwp = dw.data_ptr()
            need = lib().qg_rmsnorm_backward_workspace_bytes(rows, k)
            if need:
                ws = torch.empty(need, dtype=torch.uint8, device=dev)
                wsp = ws.data_ptr()
        rc = lib().qg_rmsnorm_backward(
            dy.data_ptr(), lddy, h.data_ptr(), ldh, code, rstd.data_ptr(), weight.data_ptr(),
            _code(weight, "weight"), rp, ldr, rows, k, dx.data_ptr(), k, dwp, wsp, need,
            _raw_stream(dev.index))
    _check(rc, "qg_rmsnorm_backward")
    return dx, dw


# ------------------------------------------------------------------ GEMM
@dataclass
class GemmFusedResult:
    out: Union[torch.Tensor, Mxfp8Result]
    checkpoint: Optional[Mxfp8Result]  # z = A . B^T + bias, for act_backward


def interleave_gate_up(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """Rows of a gate matrix and of its factor matrix in the order of
    act="swiglu": 128 gate rows, their 128 factor rows, and so on.  Done once,
    before the weights are quantised (biases: 1-D tensors work too)."""
    if gate.shape != up.shape or gate.shape[0] % GATE_COLUMNS:
        raise ValueError(f"gate and up must have one shape, rows a multiple of {GATE_COLUMNS}")
    blocks = (-1, GATE_COLUMNS) + tuple(gate.shape[1:])
    return torch.stack([gate.reshape(blocks), up.reshape(blocks)], 1).reshape(
        (2 * gate.shape[0],) + tuple(gate.shape[1:]))


def gemm_fused(a: Operand, b: Operand, bias: Optional[torch.Tensor] = None, act: str = "none",
               residual: Optional[torch.Tensor] = None, out: Union[str, torch.Tensor] = "bf16",
               layout: int = LAYOUT_MMA, checkpoint: bool = False,
               checkpoint_layout: int = LAYOUT_MMA, status: Optional[torch.Tensor] = None,
               stream: Optional[torch.cuda.Stream] = None) -> GemmFusedResult:
    """out = act(A . B^T + bias) + residual in one kernel (qg_gemm_fused), for two
    quantised operands of one format and MMA layout.  act: "none", "relu",
    "silu", "gelu" (tanh form) or "swiglu" (n columns in, n / 2 out, columns
    ordered as ``interleave_gate_up`` makes them).  out: "bf16", "f32", "mxfp8"
    (an ``Mxfp8Result`` in ``layout``, the next product's operand) or a tensor to
    write to.  checkpoint=True also returns A . B^T + bias as an ``Mxfp8Result``."""
    if type(a) is not type(b):
        raise ValueError("operands must share the format")
    if a.k != b.k or a.layout != b.layout:
        raise ValueError("operands must share K and layout")
    code = ACTIVATIONS.get(act)
    if code is None:
        raise ValueError(f"act must be one of {sorted(ACTIVATIONS)}")
    dev = _held(a, "a")
    if _held(b, "b") != dev:
        raise ValueError("operands must be on one device")
    m, n = a.rows, b.rows
    cols = n // 2 if code == ACT_SWIGLU else n
    bp = rp = ats = bts = zq = zsf = out_sf = None
    bias_code = res_code = ldr = ldc = 0
    if bias is not None:
        _vector(bias, "bias", n, dev)
        bp, bias_code = bias.data_ptr(), _code(bias, "bias")
    if residual is not None:
        ldr = _matrix(residual, "residual", m, cols, dev)
        rp, res_code = residual.data_ptr(), _code(residual, "residual")
    kind = type(a)
    fmt = FORMAT_MXFP8
    if kind is Nvfp4Result:
        fmt, ats, bts = FORMAT_NVFP4, a.tensor_scale.data_ptr(), b.tensor_scale.data_ptr()
    elif kind is Mxfp4Result:
        fmt = FORMAT_MXFP4
    with _scope(dev, stream):
        if isinstance(out, torch.Tensor):
            to, ldc = out, _matrix(out, "out", m, cols, dev)
            op, out_code = out.data_ptr(), _code(out, "out")
        elif out == "mxfp8":
            to, out_code = _new_mxfp8(m, cols, layout, dev), DTYPE_MXFP8
            op, out_sf = to.quantized.data_ptr(), to.block_scales.data_ptr()
        elif out in _TORCH:
            to, out_code = torch.empty(m, cols, dtype=_TORCH[out], device=dev), _OUTPUTS[out]
            op, ldc = to.data_ptr(), cols
        else:
            raise ValueError(f"out must be a tensor or one of {sorted(_OUTPUTS)}")
        z = None
        if checkpoint:
            z = _new_mxfp8(m, n, checkpoint_layout, dev)
            zq, zsf = z.quantized.data_ptr(), z.block_scales.data_ptr()
        e = Epilogue(code, bias_code, bp, rp, ldr, res_code, out_code, op, ldc, out_sf, zq, zsf,
                     layout, checkpoint_layout)
        rc = lib().qg_gemm_fused(
            fmt, a.quantized.data_ptr(), a.block_scales.data_ptr(), ats, b.quantized.data_ptr(),
            b.block_scales.data_ptr(), bts, m, n, a.k, a.layout, ctypes.addressof(e),
            status.data_ptr() if status is not None else None, _raw_stream(dev.index))
    _check(rc, "qg_gemm_fused")
    return GemmFusedResult(to, z)


# ------------------------------------------------------------------ backward from 8 bits
@dataclass
class ActBackwardResult:
    dz: Mxfp8Result                # [m, n], scales along n: operand of dz . W
    dz_t: Mxfp8Result              # [n, m rounded up to 32], scales along m: of dz^T . x
    dbias: Optional[torch.Tensor]  # float32 [n]


def act_backward(dout: torch.Tensor, checkpoint: Optional[Mxfp8Result], act: str,
                 layout: int = LAYOUT_MMA, want_dbias: bool = True,
                 stream: Optional[torch.cuda.Stream] = None) -> ActBackwardResult:
    """dz = dout * act'(z) from the MXFP8 checkpoint z of ``gemm_fused``,
    quantised for both gradient products, and its column sums
    (qg_act_backward_mxfp8).  dout: fp32/bf16 [m, n] ([m, n / 2] for "swiglu").
    checkpoint may be None for act="none"."""
    code = ACTIVATIONS.get(act)
    if code is None:
        raise ValueError(f"act must be one of {sorted(ACTIVATIONS)}")
    if dout.dim() != 2 or not dout.is_cuda:
        raise ValueError("dout must be a 2-D CUDA tensor")
    dev = dout.device
    m, cols = dout.shape
    n = 2 * cols if code == ACT_SWIGLU else cols
    zq = zsf = None
    z_layout = LAYOUT_MMA
    if checkpoint is not None:
        if _mxfp8(checkpoint, "checkpoint") != dev or (checkpoint.rows, checkpoint.k) != (m, n):
            raise ValueError(f"checkpoint must be {m} x {n} on {dev}")
        zq, zsf = checkpoint.quantized.data_ptr(), checkpoint.block_scales.data_ptr()
        z_layout = checkpoint.layout
    elif code != ACT_NONE:
        raise ValueError(f"act={act!r} needs the checkpoint")
    ldd = _matrix(dout, "dout", m, cols, dev)
    with _scope(dev, stream):
        dz, dz_t = _new_mxfp8(m, n, layout, dev), _new_mxfp8(n, (m + 31) // 32 * 32, layout, dev)
        db = dbp = wsp = None
        need = 0
        if want_dbias:
            db = torch.empty(n, dtype=torch.float32, device=dev)
            dbp = db.data_ptr()
            need = lib().qg_act_backward_workspace_bytes(m, n)
            if need:
                ws = torch.empty(need, dtype=torch.uint8, device=dev)
                wsp = ws.data_ptr()
        rc = lib().qg_act_backward_mxfp8(
            dout.data_ptr(), _code(dout, "dout"), ldd, zq, zsf, z_layout, code, m, n,
            dz.quantized.data_ptr(), dz.block_scales.data_ptr(), dz_t.quantized.data_ptr(),
            dz_t.block_scales.data_ptr(), layout, dbp, wsp, need, _raw_stream(dev.index))
    _check(rc, "qg_act_backward_mxfp8")
    return ActBackwardResult(dz, dz_t, db)


def transpose_mxfp8(a: Mxfp8Result, layout: int = LAYOUT_MMA,
                    stream: Optional[torch.cuda.Stream] = None) -> Mxfp8Result:
    """A's transpose (k x rows rounded up to 32, zeros beyond) requantised with
    scales along A's rows (qg_transpose_mxfp8): the kept 8-bit input of a product
    as the operand of its weight gradient."""
    dev = _mxfp8(a, "a")
    with _scope(dev, stream):
        t = _new_mxfp8(a.k, (a.rows + 31) // 32 * 32, layout, dev)
        rc = lib().qg_transpose_mxfp8(
            a.quantized.data_ptr(), a.block_scales.data_ptr(), a.layout, a.rows, a.k,
            t.quantized.data_ptr(), t.block_scales.data_ptr(), layout,
            _raw_stream(dev.index))
    _check(rc, "qg_transpose_mxfp8")
    return t
