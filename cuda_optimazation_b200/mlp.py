"""A pre-norm gated MLP block on the layer operators of ``fused.py``: forward,
backward and the single-token form.

    h   = x + residual                     one kernel: sum, RMS norm, MXFP8
    y   = rms_norm(h) * w_norm
    a   = swiglu(y . W1^T)                 one kernel: product, gate, MXFP8 (and,
                                           for training, the 8-bit checkpoint)
    out = a . W2^T + h                     one kernel: product, residual

Between the kernels the activations exist in 8 bits only; what the backward pass
keeps is y, a and the pre-activation in MXFP8 (a little over 1 byte a value),
h in the input's type and a float per row.

Command line (trains the block on a fixed random task, then decodes tokens)::

    python -m cuda_optimazation_b200.mlp [--tokens 2048] [--hidden 4096] [--inter 14336]
                                         [--steps 5]
"""
from __future__ import annotations

import argparse
import sys
import time
from dataclasses import dataclass
from typing import Optional

import torch

from . import fused, qgemm


@dataclass
class _Saved:
    y: qgemm.Mxfp8Result
    h: torch.Tensor
    rstd: torch.Tensor
    a: qgemm.Mxfp8Result
    z: qgemm.Mxfp8Result


@dataclass
class MlpGradients:
    x: torch.Tensor        # of x and of the residual alike
    norm: torch.Tensor     # float32
    gate: torch.Tensor     # float32, as the weight
    up: torch.Tensor
    down: torch.Tensor


class GatedMlp:
    """The block with fp32 master weights; quantised copies (each weight along both
    of its axes, for the product and for its input gradient) are made once a
    ``requantise()``, as a training program does after each update."""

    def __init__(self, norm: torch.Tensor, gate: torch.Tensor, up: torch.Tensor,
                 down: torch.Tensor, eps: float = 1e-5):
        inter, hidden = gate.shape
        if up.shape != gate.shape or down.shape != (hidden, inter) or norm.shape != (hidden,):
            raise ValueError("gate and up are inter x hidden, down hidden x inter, norm hidden")
        self.norm, self.gate, self.up, self.down, self.eps = norm, gate, up, down, eps
        self.requantise()

    def requantise(self) -> None:
        w1 = fused.interleave_gate_up(self.gate, self.up)
        self.w1, self.w1_t = qgemm.make_mxfp8(w1), qgemm.make_mxfp8(w1.t().contiguous())
        self.w2 = qgemm.make_mxfp8(self.down)
        self.w2_t = qgemm.make_mxfp8(self.down.t().contiguous())

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None,
                train: bool = False) -> tuple[torch.Tensor, Optional[_Saved]]:
        """The block's output (x's dtype) and, with ``train``, what ``backward`` needs."""
        n = fused.rmsnorm_mxfp8(x, self.norm, residual=residual, eps=self.eps)
        g = fused.gemm_fused(n.y, self.w1, act="swiglu", out="mxfp8", checkpoint=train)
        out = "f32" if x.dtype == torch.float32 else "bf16"
        o = fused.gemm_fused(g.out, self.w2, residual=n.h, out=out)
        return o.out, _Saved(n.y, n.h, n.rstd, g.out, g.checkpoint) if train else None

    def backward(self, dout: torch.Tensor, s: _Saved) -> MlpGradients:
        """Gradients from that of the output."""
        out = "f32" if dout.dtype == torch.float32 else "bf16"
        d = fused.act_backward(dout, None, "none", want_dbias=False)  # both 8-bit forms of dout
        da = fused.gemm_fused(d.dz, self.w2_t, out=out).out
        dw2 = fused.gemm_fused(d.dz_t, fused.transpose_mxfp8(s.a), out="f32").out
        b = fused.act_backward(da, s.z, "swiglu", want_dbias=False)
        dy = fused.gemm_fused(b.dz, self.w1_t, out=out).out
        dw1 = fused.gemm_fused(b.dz_t, fused.transpose_mxfp8(s.y), out="f32").out
        dx, dnorm = fused.rmsnorm_backward(dy, s.h, s.rstd, self.norm, dres=dout)
        pairs = dw1.view(-1, 2, fused.GATE_COLUMNS, dw1.shape[1])
        return MlpGradients(dx, dnorm, pairs[:, 0].reshape(self.gate.shape),
                            pairs[:, 1].reshape(self.up.shape), dw2)

    def step(self, g: MlpGradients, lr: float) -> None:
        """Plain gradient descent on the master weights."""
        for w, d in ((self.norm, g.norm), (self.gate, g.gate), (self.up, g.up),
                     (self.down, g.down)):
            w.sub_(d.to(w.dtype), alpha=lr)
        self.requantise()


def random_block(hidden: int, inter: int, seed: int = 0, device="cuda") -> GatedMlp:
    g = torch.Generator(device=device).manual_seed(seed)

    def rand(*shape, std):
        return torch.randn(*shape, generator=g, device=device) * std

    return GatedMlp(1 + rand(hidden, std=0.1), rand(inter, hidden, std=hidden ** -0.5),
                    rand(inter, hidden, std=hidden ** -0.5), rand(hidden, inter, std=inter ** -0.5))


def main(argv: Optional[list[str]] = None) -> int:
    ap = argparse.ArgumentParser(prog="python -m cuda_optimazation_b200.mlp")
    ap.add_argument("--tokens", type=int, default=2048)
    ap.add_argument("--hidden", type=int, default=4096)
    ap.add_argument("--inter", type=int, default=14336)
    ap.add_argument("--steps", type=int, default=5)
    args = ap.parse_args(argv)
    block, target = random_block(args.hidden, args.inter), random_block(args.hidden, args.inter, 1)
    x = torch.randn(args.tokens, args.hidden, device="cuda").to(torch.bfloat16)
    want = target.forward(x)[0].float()
    for i in range(args.steps):
        torch.cuda.synchronize()
        t = time.perf_counter()
        out, saved = block.forward(x, train=True)
        err = out.float() - want
        grads = block.backward((err / args.tokens).to(torch.bfloat16), saved)
        torch.cuda.synchronize()
        ms = (time.perf_counter() - t) * 1e3
        print(f"step {i}: loss {float(err.square().sum()) / (2 * args.tokens):.4f}  "
              f"forward and backward {ms:.2f} ms")
        block.step(grads, 0.5)
    token = x[:1].contiguous()
    block.forward(token)
    torch.cuda.synchronize()
    t = time.perf_counter()
    for _ in range(100):
        block.forward(token)
    torch.cuda.synchronize()
    print(f"one token: {(time.perf_counter() - t) * 1e4:.1f} us")
    return 0


if __name__ == "__main__":
    sys.exit(main())
