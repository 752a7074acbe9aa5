"""CPU: the layer operators refuse bad arguments before any CUDA call (fake
addresses are never dereferenced)."""
import ctypes

import pytest
import torch

A, MIS = 4096, 4104  # a 16-byte aligned fake address and one that is not
BIG = 1 << 40


def norm(L, x=A, dt=1, ldx=256, res=A, ldr=256, w=A, wdt=1, eps=1e-5, rows=4, k=256, layout=1,
         q=A, sf=A, h=A, ldh=256, rstd=A):
    return L.qg_rmsnorm_mxfp8(x, dt, ldx, res, ldr, w, wdt, eps, rows, k, layout, q, sf, h, ldh,
                              rstd, None)


def test_rmsnorm_refusals(qlib):
    L = qlib.lib()
    for bad in ("x", "w", "q", "sf"):
        assert norm(L, **{bad: None}) == qlib.ERR_ARG
    assert norm(L, eps=-1.0) == qlib.ERR_ARG
    assert norm(L, eps=float("nan")) == qlib.ERR_ARG
    assert norm(L, dt=2) == qlib.ERR_DTYPE
    assert norm(L, wdt=7) == qlib.ERR_DTYPE
    assert norm(L, layout=3) == qlib.ERR_LAYOUT
    for bad in (dict(rows=0), dict(k=48), dict(k=0), dict(k=65536, ldx=65536, ldr=65536, ldh=65536),
                dict(ldx=255), dict(ldr=128), dict(ldh=0), dict(rows=1 << 31)):
        assert norm(L, **bad) == qlib.ERR_SHAPE, bad
    for bad in (dict(x=MIS), dict(res=MIS), dict(h=MIS), dict(w=MIS), dict(q=MIS), dict(ldx=257),
                dict(ldr=260), dict(ldh=258), dict(sf=A + 2), dict(rstd=A + 2)):
        assert norm(L, **bad) == qlib.ERR_ALIGN, bad


def norm_bwd(L, dy=A, lddy=256, h=A, ldh=256, dt=0, rstd=A, w=A, wdt=0, dres=None, lddres=0,
             rows=600, k=256, dx=2 * A, lddx=256, dw=A, ws=A, wsb=BIG):
    return L.qg_rmsnorm_backward(dy, lddy, h, ldh, dt, rstd, w, wdt, dres, lddres, rows, k, dx,
                                 lddx, dw, ws, wsb, None)


def test_rmsnorm_backward_refusals(qlib):
    L = qlib.lib()
    for bad in ("dy", "h", "rstd", "w", "dx", "ws"):
        assert norm_bwd(L, **{bad: None}) == qlib.ERR_ARG, bad
    assert norm_bwd(L, dx=A) == qlib.ERR_ARG  # dy's own buffer
    need = L.qg_rmsnorm_backward_workspace_bytes(600, 256)
    assert need > 0 and need % (256 * 4) == 0
    assert L.qg_rmsnorm_backward_workspace_bytes(0, 256) == 0
    assert L.qg_rmsnorm_backward_workspace_bytes(4, 256) == 0  # few rows join by themselves
    assert norm_bwd(L, wsb=need - 1) == qlib.ERR_ARG
    assert norm_bwd(L, dt=3) == qlib.ERR_DTYPE
    for bad in (dict(rows=0), dict(k=40), dict(lddy=8), dict(ldh=8), dict(lddx=8),
                dict(dres=A, lddres=8)):
        assert norm_bwd(L, **bad) == qlib.ERR_SHAPE, bad
    for bad in (dict(dy=MIS), dict(h=MIS), dict(dx=A + 8 * 1001), dict(w=MIS), dict(ws=MIS), dict(lddx=257),
                dict(dres=MIS, lddres=256), dict(dw=A + 1)):
        assert norm_bwd(L, **bad) == qlib.ERR_ALIGN, bad


def gemm(qlib, fmt=0, a=A, b=A, m=64, n=256, k=128, sf_layout=1, **epi):
    e = qlib.Epilogue()
    fields = dict(act=0, out=A, out_dtype=1, ldc=256) | epi
    for name, v in fields.items():
        setattr(e, name, v)
    return qlib.lib().qg_gemm_fused(fmt, a, A, None, b, A, None, m, n, k, sf_layout,
                                    ctypes.addressof(e), None, None)


def test_gemm_refusals(qlib):
    L = qlib.lib()
    assert L.qg_gemm_fused(0, A, A, None, A, A, None, 64, 256, 128, 1, None, None,
                           None) == qlib.ERR_ARG
    assert gemm(qlib, out=None) == qlib.ERR_ARG
    assert gemm(qlib, act=5) == qlib.ERR_ARG
    assert gemm(qlib, a=None) == qlib.ERR_ARG
    assert gemm(qlib, out_dtype=2) == qlib.ERR_ARG  # no scales
    assert gemm(qlib, ckpt_q=A) == qlib.ERR_ARG
    for bad in (dict(fmt=3), dict(out_dtype=4), dict(bias=A, bias_dtype=2),
                dict(residual=A, residual_dtype=2, ldr=256)):
        assert gemm(qlib, **bad) == qlib.ERR_DTYPE, bad
    for bad in (dict(sf_layout=0), dict(out_dtype=2, out_sf=A, out_layout=3),
                dict(ckpt_q=A, ckpt_sf=A, ckpt_layout=-1)):
        assert gemm(qlib, **bad) == qlib.ERR_LAYOUT, bad
    for bad in (dict(m=0), dict(n=0), dict(k=48), dict(ldc=255), dict(act=4, n=128, ldc=128),
                dict(n=40, out_dtype=2, out_sf=A), dict(n=40, ckpt_q=A, ckpt_sf=A),
                dict(residual=A, ldr=255), dict(m=1 << 31)):
        assert gemm(qlib, **bad) == qlib.ERR_SHAPE, bad
    for bad in (dict(a=MIS), dict(out=A + 1), dict(out_dtype=2, out=MIS, out_sf=A),
                dict(out_dtype=2, out_sf=MIS), dict(ckpt_q=MIS, ckpt_sf=A),
                dict(bias=A + 2, bias_dtype=0), dict(residual=A + 1, residual_dtype=1, ldr=256)):
        assert gemm(qlib, **bad) == qlib.ERR_ALIGN, bad


def act_bwd(L, d=A, dt=1, ldd=256, zq=A, zsf=A, zl=1, act=2, m=2000, n=256, dz=A, dzs=A, t=A, ts=A,
            lay=1, db=A, ws=A, wsb=BIG):
    return L.qg_act_backward_mxfp8(d, dt, ldd, zq, zsf, zl, act, m, n, dz, dzs, t, ts, lay, db, ws,
                                   wsb, None)


def test_act_backward_refusals(qlib):
    L = qlib.lib()
    for bad in ("d", "zq", "zsf", "dz", "dzs", "t", "ts", "ws"):
        assert act_bwd(L, **{bad: None}) == qlib.ERR_ARG, bad
    assert act_bwd(L, act=5) == qlib.ERR_ARG
    assert act_bwd(L, wsb=L.qg_act_backward_workspace_bytes(2000, 256) - 1) == qlib.ERR_ARG
    assert L.qg_act_backward_workspace_bytes(64, 256) == 0  # one row tile
    assert act_bwd(L, dt=2) == qlib.ERR_DTYPE
    for bad in (dict(zl=3), dict(lay=0), dict(lay=3)):
        assert act_bwd(L, **bad) == qlib.ERR_LAYOUT, bad
    for bad in (dict(m=0), dict(n=48), dict(act=4, n=128), dict(ldd=255)):
        assert act_bwd(L, **bad) == qlib.ERR_SHAPE, bad
    for bad in (dict(d=MIS), dict(zq=MIS), dict(dz=MIS), dict(dzs=MIS), dict(t=MIS), dict(ts=MIS),
                dict(ldd=257), dict(db=A + 2), dict(ws=MIS)):
        assert act_bwd(L, **bad) == qlib.ERR_ALIGN, bad


def test_transpose_refusals(qlib):
    L = qlib.lib()
    ok = [A, A, 1, 64, 256, A, A, 1, None]

    def call(**at):
        args = list(ok)
        for i, v in at.items():
            args[int(i[1:])] = v
        return L.qg_transpose_mxfp8(*args)

    for i in (0, 1, 5, 6):
        assert call(**{f"_{i}": None}) == qlib.ERR_ARG
    assert call(_2=3) == qlib.ERR_LAYOUT and call(_7=0) == qlib.ERR_LAYOUT
    assert call(_3=0) == qlib.ERR_SHAPE and call(_4=40) == qlib.ERR_SHAPE
    for i in (0, 5, 6):
        assert call(**{f"_{i}": MIS}) == qlib.ERR_ALIGN


def test_wrapper_refusals(qlib):
    from cuda_optimazation_b200 import fused
    x, w = torch.zeros(4, 64), torch.zeros(64)
    with pytest.raises(ValueError):
        fused.rmsnorm_mxfp8(x, w)  # not a CUDA tensor
    with pytest.raises(ValueError):
        fused.rmsnorm_backward(x, x, torch.zeros(4), w)
    with pytest.raises(ValueError):
        fused.act_backward(x, None, "none")
    with pytest.raises(ValueError):
        fused.act_backward(x, None, "tanh")
    z = qlib.Mxfp8Result(torch.zeros(256, dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8),
                         4, 64, 1)
    with pytest.raises(ValueError):
        fused.transpose_mxfp8(z)
    with pytest.raises(TypeError):
        fused.transpose_mxfp8(x)
    with pytest.raises(ValueError):
        fused.gemm_fused(z, z)
    with pytest.raises(ValueError):
        fused.gemm_fused(z, z, act="tanh")
    short = qlib.Mxfp8Result(z.quantized[:100], z.block_scales, 4, 64, 1)
    with pytest.raises(ValueError):
        fused.gemm_fused(short, z)
    with pytest.raises(ValueError):
        fused.interleave_gate_up(torch.zeros(100, 4), torch.zeros(100, 4))
