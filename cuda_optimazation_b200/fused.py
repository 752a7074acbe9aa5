"""Layer operators around the block-scaled GEMM, over the C ABI in
include/qgemm.h: what a transformer layer computes next to its products,
writing and reading the operands that the products use.

``rmsnorm_mxfp8`` (RMS norm, residual addition, 8-bit output) and
``rmsnorm_backward``; ``gemm_fused`` (bias, activation, residual in the GEMM's
epilogue, 8-bit output, 8-bit checkpoint of the pre-activation);
``act_backward`` and ``transpose_mxfp8`` (the checkpoint and the kept 8-bit
input in the backward pass).  ``mlp.py`` runs them together.

Arguments are checked and outputs allocated, on the stream that the operator is
launched on (``stream``, by default the current one), in
csrc/torch_binding.cpp: a call on a decode step's sizes costs the host about as
much as the GPU.  A missing binding raises; there is no fallback.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Union

import torch

from .qgemm import (
    ACT_GELU, ACT_NONE, ACT_RELU, ACT_SILU, ACT_SWIGLU, DTYPE_BF16, DTYPE_F32, DTYPE_MXFP8,
    FORMAT_MXFP4, FORMAT_MXFP8, FORMAT_NVFP4, LAYOUT_MMA, Mxfp4Result, Mxfp8Result, Nvfp4Result,
    QGemmError, lib,
)

ACTIVATIONS = {"none": ACT_NONE, "relu": ACT_RELU, "silu": ACT_SILU, "gelu": ACT_GELU,
               "swiglu": ACT_SWIGLU}
GATE_COLUMNS = 128  # columns of a gate block of the gated activation
_OUTPUTS = {"f32": DTYPE_F32, "bf16": DTYPE_BF16, "mxfp8": DTYPE_MXFP8}
_FORMATS = {Mxfp8Result: FORMAT_MXFP8, Nvfp4Result: FORMAT_NVFP4, Mxfp4Result: FORMAT_MXFP4}

Operand = Union[Mxfp8Result, Nvfp4Result, Mxfp4Result]

_module = None


def _native():
    """The binding module (raises if it has not been built)."""
    global _module
    if _module is None:
        lib()
        try:
            from . import _binding
        except ImportError as e:
            raise RuntimeError("the torch binding is missing: build it with "
                               "`python -m cuda_optimazation_b200.build`") from e
        _module = _binding
    return _module


def _act_code(act: str) -> int:
    code = ACTIVATIONS.get(act)
    if code is None:
        raise ValueError(f"act must be one of {sorted(ACTIVATIONS)}")
    return code


def _on(stream: torch.cuda.Stream, held) -> torch.cuda.StreamContext:
    """`stream` as the current one for a call on `held` (a matrix or an operand)."""
    device = getattr(getattr(held, "quantized", held), "device", None)
    if device is not None and device != stream.device:
        raise ValueError(f"stream is on {stream.device}, the operands on {device}")
    return torch.cuda.stream(stream)


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
    if stream is not None:
        with _on(stream, x):
            return rmsnorm_mxfp8(x, weight, residual, eps, layout, h)
    rc, q, sf, new_h, rstd = _native().rmsnorm_mxfp8(x, weight, residual, eps, layout, h)
    if rc:
        raise QGemmError(rc, "qg_rmsnorm_mxfp8")
    if h is None:
        h = x if new_h is None else new_h
    return RmsNormResult(Mxfp8Result(q, sf, x.shape[0], x.shape[1], layout), h, rstd)


def rmsnorm_backward(dy: torch.Tensor, h: torch.Tensor, rstd: torch.Tensor, weight: torch.Tensor,
                     dres: Optional[torch.Tensor] = None, want_dweight: bool = True,
                     stream: Optional[torch.cuda.Stream] = None
                     ) -> tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Gradient of ``rmsnorm_mxfp8`` (the quantisation passed straight through):
    (dx, dweight) from dy = dL/dy, the saved h and rstd, and optionally dres,
    the gradient that reaches h past the norm.  dx (h's dtype) is the gradient
    of x and of the residual; dweight is fp32 (None if not wanted)."""
    if stream is not None:
        with _on(stream, dy):
            return rmsnorm_backward(dy, h, rstd, weight, dres, want_dweight)
    rc, dx, dw = _native().rmsnorm_backward(dy, h, rstd, weight, dres, want_dweight)
    if rc:
        raise QGemmError(rc, "qg_rmsnorm_backward")
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
    if stream is not None:
        with _on(stream, a):
            return gemm_fused(a, b, bias, act, residual, out, layout, checkpoint,
                              checkpoint_layout, status)
    fmt = _FORMATS.get(type(a))
    if fmt is None or type(a) is not type(b):
        raise ValueError("operands must be quantised and share the format")
    if a.k != b.k or a.layout != b.layout:
        raise ValueError("operands must share K and layout")
    code = _act_code(act)
    given = None
    if isinstance(out, str):
        kind = _OUTPUTS.get(out)
        if kind is None:
            raise ValueError(f"out must be a tensor or one of {sorted(_OUTPUTS)}")
    else:
        kind, given = DTYPE_F32, out
    ats, bts = (a.tensor_scale, b.tensor_scale) if fmt == FORMAT_NVFP4 else (None, None)
    m, n = a.rows, b.rows
    rc, o, osf, zq, zsf = _native().gemm_fused(
        fmt, a.quantized, a.block_scales, ats, m, b.quantized, b.block_scales, bts, n, a.k,
        a.layout, bias, code, residual, kind, given, layout, checkpoint, checkpoint_layout, status)
    if rc:
        raise QGemmError(rc, "qg_gemm_fused")
    if kind == DTYPE_MXFP8:
        o = Mxfp8Result(o, osf, m, n // 2 if code == ACT_SWIGLU else n, layout)
    elif given is not None:
        o = given
    return GemmFusedResult(
        o, None if zq is None else Mxfp8Result(zq, zsf, m, n, checkpoint_layout))


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
    if stream is not None:
        with _on(stream, dout):
            return act_backward(dout, checkpoint, act, layout, want_dbias)
    code = _act_code(act)
    z = checkpoint
    if z is None:
        if code != ACT_NONE:
            raise ValueError(f"act={act!r} needs the checkpoint")
        rc, q, sf, tq, tsf, db = _native().act_backward(dout, None, None, 0, 0, LAYOUT_MMA, code,
                                                        layout, want_dbias)
    else:
        if type(z) is not Mxfp8Result:
            raise TypeError("checkpoint must be an Mxfp8Result")
        rc, q, sf, tq, tsf, db = _native().act_backward(
            dout, z.quantized, z.block_scales, z.rows, z.k, z.layout, code, layout, want_dbias)
    if rc:
        raise QGemmError(rc, "qg_act_backward_mxfp8")
    m, n = dout.shape
    if code == ACT_SWIGLU:
        n *= 2
    return ActBackwardResult(Mxfp8Result(q, sf, m, n, layout),
                             Mxfp8Result(tq, tsf, n, (m + 31) // 32 * 32, layout), db)


def transpose_mxfp8(a: Mxfp8Result, layout: int = LAYOUT_MMA,
                    stream: Optional[torch.cuda.Stream] = None) -> Mxfp8Result:
    """A's transpose (k x rows rounded up to 32, zeros beyond) requantised with
    scales along A's rows (qg_transpose_mxfp8): the kept 8-bit input of a product
    as the operand of its weight gradient."""
    if stream is not None:
        with _on(stream, a):
            return transpose_mxfp8(a, layout)
    if type(a) is not Mxfp8Result:
        raise TypeError("a must be an Mxfp8Result")
    rc, q, sf = _native().transpose_mxfp8(a.quantized, a.block_scales, a.rows, a.k, a.layout,
                                          layout)
    if rc:
        raise QGemmError(rc, "qg_transpose_mxfp8")
    return Mxfp8Result(q, sf, a.k, (a.rows + 31) // 32 * 32, layout)
