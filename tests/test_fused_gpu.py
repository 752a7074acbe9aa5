"""GPU: the layer operators against their definitions in 64 bits.

Tolerances: a sum of fp32 values in the kernels runs over at most a few hundred
sequential additions, so it is good to 2^-16 of the sum of magnitudes; the
GEMM's accumulation (K / 32 groups, K < 4096) to 2^-16 of sum |a b|; outputs add
half a step of their type."""
import math

import pytest
import torch

import fused_ref as R

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
F64 = torch.float64
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
# Half a step relative to the value: 2^-p for p significant bits (8 and 24).
STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


@pytest.fixture(scope="module")
def F(qlib):
    from cuda_optimazation_b200 import fused
    return fused


def rand(*shape, seed=0, std=1.0, dtype=torch.float32, pad=0):
    g = torch.Generator(device=DEV).manual_seed(seed * 7919 + sum(shape))
    full = shape[:-1] + (shape[-1] + pad,)
    return (torch.randn(*full, generator=g, device=DEV) * std).to(dtype)[..., :shape[-1]]


def close(got, ref, tol):
    assert got.shape == ref.shape
    err = (got.to(F64) - ref).abs()
    assert bool((err <= tol).all()), f"worst excess {float((err - tol).max()):.3e}"


# ------------------------------------------------------------------ RMS norm
NORM = [(1, 32), (1, 8192), (3, 96), (127, 160), (128, 4096), (129, 5152), (300, 64), (2, 16416),
        (5, 32768), (1000, 1024), (14171, 640), (5000, 2048), (1500, 8192), (700, 13056),
        (400, 16384), (600, 32768)]


@pytest.mark.parametrize("rows,k", NORM)
@pytest.mark.parametrize("xt,wt", [("bf16", "bf16"), ("f32", "f32"), ("bf16", "f32"),
                                   ("f32", "bf16")])
def test_norm(F, rows, k, xt, wt):
    layout = (rows + k // 32) % 3
    pad = 8 if rows % 2 else 0
    x = rand(rows, k, seed=1, dtype=TYPES[xt], pad=pad)
    res = rand(rows, k, seed=2, std=3.0, dtype=TYPES[xt]) if k != 64 else None
    w = rand(k, seed=3, dtype=TYPES[wt])
    o = F.rmsnorm_mxfp8(x, w, residual=res, eps=1e-5, layout=layout)
    h, rstd, y = R.norm(x, res, w, 1e-5)
    close(o.rstd, rstd, 2.0 ** -16 * rstd)
    if res is None:
        assert o.h is x
    else:
        close(o.h, h, STEP[x.dtype] * 1.01 * h.abs())
    assert (o.y.rows, o.y.k, o.y.layout) == (rows, k, layout)
    R.check_mx(o.y, y, 2.0 ** -15 * y.abs())


def test_norm_special_rows(F):
    """A row of zeros, one with a NaN, one with an infinity, one of tiny values:
    each stays in its row, and zeros get the zero block's code."""
    x = rand(6, 256, seed=4)
    x[1] = 0
    x[2, 5] = float("nan")
    x[3, 7] = float("inf")
    x[4] *= 1e-30
    w = torch.ones(256, device=DEV)
    o = F.rmsnorm_mxfp8(x, w, eps=0.5)
    q, e = R.parts(o.y)
    assert bool((q[1] == 0).all()) and bool((e[1] == -127).all())
    assert bool(torch.isnan(q[2]).all())
    assert bool((q[3, :7] == 0).all()) and bool(torch.isnan(q[3, 7]))
    _, rstd, y = R.norm(x, None, w, 0.5)
    keep = [0, 1, 4, 5]
    close(o.rstd[keep], rstd[keep], 2.0 ** -16 * rstd[keep])
    clean = F.rmsnorm_mxfp8(x[keep].contiguous(), w, eps=0.5)
    assert torch.equal(o.y.quantized.view(6, 256)[keep], clean.y.quantized.view(4, 256))


def test_norm_in_place_and_side_stream(F):
    rows, k = 200, 2048
    x, res = (rand(rows, k, seed=s, dtype=torch.bfloat16) for s in (5, 6))
    w = rand(k, seed=7)
    want = F.rmsnorm_mxfp8(x, w, residual=res)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    into = res.clone()
    side.wait_stream(torch.cuda.current_stream())
    got = F.rmsnorm_mxfp8(x, w, residual=into, h=into, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert got.h is into and torch.equal(into, want.h)
    assert torch.equal(got.y.quantized, want.y.quantized)
    assert torch.equal(got.y.block_scales, want.y.block_scales)


@pytest.mark.parametrize("rows,k", NORM + [(700, 512)])
@pytest.mark.parametrize("xt,wt", [("bf16", "bf16"), ("f32", "f32"), ("f32", "bf16")])
def test_norm_backward(F, rows, k, xt, wt):
    h = rand(rows, k, seed=11, std=2.0, dtype=TYPES[xt], pad=8 if rows % 2 else 0)
    dy = rand(rows, k, seed=12, std=0.1, dtype=TYPES[xt])
    dres = rand(rows, k, seed=13, std=0.1, dtype=TYPES[xt]) if k % 64 == 0 else None
    w = rand(k, seed=14, dtype=TYPES[wt])
    rstd = (h.float().square().mean(-1) + 1e-5).rsqrt()
    dx, dw = F.rmsnorm_backward(dy, h, rstd, w, dres=dres)
    r = rstd.to(F64)[:, None]
    xh, g = h.to(F64) * r, dy.to(F64) * w.to(F64)
    c = (g * xh).mean(-1, keepdim=True)
    ref = r * (g - xh * c)
    size = r * (g.abs() + xh.abs() * ((g * xh).abs().mean(-1, keepdim=True)))
    if dres is not None:
        ref = ref + dres.to(F64)
        size = size + dres.to(F64).abs()
    close(dx, ref, 2.0 ** -16 * size + 1.01 * STEP[h.dtype] * ref.abs())
    prod = dy.to(F64) * xh
    close(dw, prod.sum(0), 2.0 ** -16 * prod.abs().sum(0))
    again, dw2 = F.rmsnorm_backward(dy, h, rstd, w, dres=dres)
    assert torch.equal(dx, again) and torch.equal(dw, dw2), "not deterministic"
    only, none = F.rmsnorm_backward(dy, h, rstd, w, dres=dres, want_dweight=False)
    assert none is None and torch.equal(only, dx)


def test_norm_backward_against_differences(F):
    """dx and dweight against central differences of sum(dy * y) in 64 bits:
    the step's error is of order step^2 = 1e-8 of the third derivative."""
    rows, k, step = 3, 64, 1e-4
    h, dy, w = rand(rows, k, seed=21), rand(rows, k, seed=22), rand(k, seed=23)
    rstd = (h.float().square().mean(-1) + 1e-5).rsqrt()
    dx, dw = F.rmsnorm_backward(dy, h, rstd, w)

    def loss(hh, ww):
        return (dy.to(F64) * R.norm(hh, None, ww, 1e-5)[2]).sum()

    for i, j in [(0, 0), (1, 17), (2, 63), (2, 32)]:
        d = torch.zeros(rows, k, dtype=F64, device=DEV)
        d[i, j] = step
        num = (loss(h.to(F64) + d, w) - loss(h.to(F64) - d, w)) / (2 * step)
        assert abs(float(num) - float(dx[i, j])) <= 1e-5 * (1 + abs(float(num)))
        num = (loss(h, w.to(F64) + d[i]) - loss(h, w.to(F64) - d[i])) / (2 * step)
        assert abs(float(num) - float(dw[j])) <= 1e-5 * (1 + abs(float(num)))


# ------------------------------------------------------------------ GEMM
def operand(qlib, rows, k, fmt, seed, std=1.0, layout=1):
    """(operand, its exact 64-bit value), quantised by the library."""
    x = rand(rows, k, seed=seed, std=std)
    if fmt == "mxfp8":
        r = qlib.make_mxfp8(x, layout)
        return r, R.value(r)
    make = qlib.make_nvfp4 if fmt == "nvfp4" else qlib.make_mxfp4
    r = make(x, layout)
    table = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, 0, -.5, -1, -1.5, -2, -3, -4, -6], dtype=F64,
                         device=DEV)
    p = r.quantized.view(rows, k // 2)
    v = table[torch.stack([p & 15, p >> 4], -1).long()].view(rows, k)
    sv = 16 if fmt == "nvfp4" else 32
    at, _ = R.chunk_order(rows, k // sv, layout)
    codes = r.block_scales[at.to(DEV)]
    s = (codes.view(R.E4M3).to(F64) if fmt == "nvfp4" else torch.exp2(codes.to(F64) - 127))
    v = (v.view(rows, k // sv, sv) * s.unsqueeze(-1)).view(rows, k)
    return r, v * r.tensor_scale.to(F64) if fmt == "nvfp4" else v


def gemm_case(F, qlib, m, n, k, fmt="mxfp8", act="none", out="bf16", bias=None, res=None,
              ckpt=False, layout=1, sf_layout=1, ckpt_layout=1):
    a, av = operand(qlib, m, k, fmt, 31, layout=sf_layout)
    b, bv = operand(qlib, n, k, fmt, 32, 1.0 / math.sqrt(k), layout=sf_layout)
    cols = n // 2 if act == "swiglu" else n
    bt = rand(n, seed=33, dtype=TYPES[bias]) if bias else None
    rt = rand(m, cols, seed=34, std=2.0, dtype=TYPES[res], pad=3) if res else None
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    o = F.gemm_fused(a, b, bias=bt, act=act, residual=rt, out=out, layout=layout,
                     checkpoint=ckpt, checkpoint_layout=ckpt_layout, status=status)
    rc, code = qlib.read_status(status)
    assert rc == qlib.OK, f"device status {code}"
    z = av @ bv.t()
    tol = 2.0 ** -16 * (av.abs() @ bv.abs().t())
    if bt is not None:
        z = z + bt.to(F64)
        tol = tol + 2.0 ** -22 * bt.to(F64).abs()
    y, ty = R.act(z, act), R.act_tol(z, tol, act)
    if rt is not None:
        y = y + rt.to(F64)
        ty = ty + 2.0 ** -22 * rt.to(F64).abs()
    if out == "mxfp8":
        assert (o.out.rows, o.out.k, o.out.layout) == (m, cols, layout)
        R.check_mx(o.out, y, ty)
    else:
        assert o.out.dtype == TYPES[out]
        close(o.out, y, ty + 1.01 * STEP[o.out.dtype] * y.abs())
    if ckpt:
        assert (o.checkpoint.rows, o.checkpoint.k, o.checkpoint.layout) == (m, n, ckpt_layout)
        R.check_mx(o.checkpoint, z, tol)
    else:
        assert o.checkpoint is None


# Rows from one to several tiles, odd sizes against the 256 x 256 tiles, K below
# and across a 128-byte stage.
SHAPES = [(1, 256, 32), (1, 4096, 2048), (2, 33, 96), (7, 512, 4000), (16, 1000, 512),
          (33, 256, 160), (64, 768, 1024), (128, 512, 256), (129, 300, 64), (256, 256, 256),
          (257, 513, 544), (600, 1030, 1056)]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("fmt", ["mxfp8", "nvfp4", "mxfp4"])
def test_gemm_shapes(F, qlib, m, n, k, fmt):
    gemm_case(F, qlib, m, n, k, fmt, act="gelu", bias="f32", res="bf16",
              out="bf16" if n % 2 else "f32")


@pytest.mark.parametrize("m,n", [(150, 1959), (300, 70), (257, 8)])
@pytest.mark.parametrize("res", [None, "bf16", "f32"])
@pytest.mark.parametrize("out", ["bf16", "f32"])
def test_gemm_odd_rows(F, qlib, m, n, res, out):
    """Rows whose starts 16-byte accesses cannot use."""
    gemm_case(F, qlib, m, n, 96, act="silu", bias="bf16", res=res, out=out)


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "swiglu"])
@pytest.mark.parametrize("out", ["bf16", "f32", "mxfp8"])
@pytest.mark.parametrize("m", [1, 20, 100, 300])
def test_gemm_activations(F, qlib, m, act, out):
    gemm_case(F, qlib, m, 512, 320, act=act, out=out, bias="bf16", res="f32", ckpt=True,
              layout=m % 3, ckpt_layout=(m + 1) % 3)


@pytest.mark.parametrize("fmt", ["mxfp8", "nvfp4", "mxfp4"])
@pytest.mark.parametrize("m,n", [(1, 256), (5, 1280), (130, 768)])
def test_gemm_gated(F, qlib, m, n, fmt):
    gemm_case(F, qlib, m, n, 512, fmt, act="swiglu", out="mxfp8", ckpt=True, sf_layout=2)


@pytest.mark.parametrize("m,n", [(1, 32), (9, 96), (40, 224), (200, 416)])
def test_gemm_ragged_blocks(F, qlib, m, n):
    """MXFP8 outputs whose last scale chunk is part padding."""
    gemm_case(F, qlib, m, n, 128, out="mxfp8", ckpt=True, res="bf16", ckpt_layout=2)


def test_gemm_long_k_and_residual_in_place(F, qlib):
    a, av = operand(qlib, 96, 3968, "mxfp8", 41)
    b, bv = operand(qlib, 640, 3968, "mxfp8", 42, 0.02)
    c = rand(96, 640, seed=43, dtype=torch.bfloat16)
    ref = av @ bv.t() + c.to(F64)
    tol = 2.0 ** -16 * (av.abs() @ bv.abs().t()) + 2.0 ** -8 * ref.abs()
    o = F.gemm_fused(a, b, residual=c, out=c)
    assert o.out is c
    close(c, ref, tol)


@pytest.mark.parametrize("m,n", [(300, 768), (260, 601)])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_gemm_over_its_residual(F, qlib, m, n, dt):
    """Several tiles, rows on 16 bytes and odd ones, written over the residual."""
    a, av = operand(qlib, m, 256, "mxfp8", 45)
    b, bv = operand(qlib, n, 256, "mxfp8", 46, 0.06)
    c = rand(m, n, seed=47, dtype=TYPES[dt])
    ref = av @ bv.t() + c.to(F64)
    tol = 2.0 ** -16 * (av.abs() @ bv.abs().t()) + 1.01 * STEP[c.dtype] * ref.abs()
    tol = tol + 2.0 ** -22 * c.to(F64).abs()
    assert F.gemm_fused(a, b, residual=c, out=c).out is c
    close(c, ref, tol)


def test_gemm_matches_plain_gemm(F, qlib):
    """Without an epilogue the product is the plain GEMM's."""
    for m in (300, 1024):
        a, _ = operand(qlib, m, 1024, "mxfp8", 51)
        b, _ = operand(qlib, 768, 1024, "mxfp8", 52)
        want = qlib.block_scaled_gemm(a, b, torch.float32)
        assert torch.equal(F.gemm_fused(a, b, out="f32").out, want)


def test_gemm_repeats_and_streams(F, qlib):
    a, _ = operand(qlib, 8, 2048, "mxfp8", 61)
    b, _ = operand(qlib, 1024, 2048, "mxfp8", 62)
    want = F.gemm_fused(a, b, act="silu").out
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = [F.gemm_fused(a, b, act="silu", stream=side).out for _ in range(4)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(o, want) for o in outs)


def test_gemm_special_values(F, qlib):
    """An infinite and a NaN residual or bias stay in their element, column or block."""
    a, _ = operand(qlib, 40, 256, "mxfp8", 71)
    b, _ = operand(qlib, 256, 256, "mxfp8", 72)
    clean = F.gemm_fused(a, b, out="f32").out
    res = torch.zeros(40, 256, device=DEV)
    res[3, 100], res[4, 101] = float("inf"), float("nan")
    got = F.gemm_fused(a, b, residual=res, out="f32").out
    assert bool(torch.isinf(got[3, 100])) and bool(torch.isnan(got[4, 101]))
    keep = torch.isfinite(got)
    assert int((~keep).sum()) == 2 and torch.equal(got[keep], clean[keep])
    q, _ = R.parts(F.gemm_fused(a, b, residual=res, out="mxfp8").out)
    assert bool(torch.isnan(q[4, 101])) and int(torch.isnan(q).sum()) == 1
    assert float(q[3, 100]) == 448.0
    bias = torch.zeros(256, device=DEV)
    bias[7] = float("nan")
    got = F.gemm_fused(a, b, bias=bias, act="relu", out="f32").out
    assert bool(torch.isnan(got[:, 7]).all()) and int(torch.isnan(got).sum()) == 40


def test_interleave(F):
    g, u = rand(256, 8, seed=81), rand(256, 8, seed=82)
    w = F.interleave_gate_up(g, u)
    assert torch.equal(w[:128], g[:128]) and torch.equal(w[128:256], u[:128])
    assert torch.equal(w[256:384], g[128:]) and torch.equal(w[384:], u[128:])
    assert torch.equal(F.interleave_gate_up(g[:, 0], u[:, 0]), w[:, 0])


# ------------------------------------------------------------------ backward from 8 bits
def act_grad(d, z, name):
    """dz by the activation's derivative (from autograd, in 64 bits)."""
    z = z.clone().requires_grad_(True)
    R.act(z, name).backward(d)
    return z.grad


ACT_SHAPES = [(1, 256), (2, 512), (31, 256), (32, 768), (100, 256), (128, 512), (333, 1024)]


@pytest.mark.parametrize("m,n", ACT_SHAPES + [(5, 32), (130, 96), (257, 416)])
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "swiglu"])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_act_backward(F, qlib, m, n, act, dt):
    if act == "swiglu" and n % 256:
        pytest.skip("the gated form takes whole gate blocks")
    cols = n // 2 if act == "swiglu" else n
    layout, z_layout = 1 + m % 2, (m + n // 32) % 3
    z = qlib.make_mxfp8(rand(m, n, seed=91, std=2.0), z_layout)
    zv = R.value(z)
    d = rand(m, cols, seed=92, std=0.01, dtype=TYPES[dt], pad=8 if m % 2 else 0)
    o = F.act_backward(d, z if act != "none" or m % 2 else None, act, layout=layout)
    dz = d.to(F64) if act == "none" else act_grad(d.to(F64), zv, act)
    if act == "swiglu":
        g, u = zv.view(m, -1, 2, 128).unbind(2)
        dd = d.to(F64).view(m, -1, 128)
        tol = torch.stack([(dd * u).abs(), (dd * g).abs()], 2).reshape(m, n) * 2.0 ** -19
        tol = tol * (1 + zv.abs())
    else:
        tol = 2.0 ** -19 * d.to(F64).abs() * (1 + zv.abs())
        if act in ("none", "relu"):
            tol = 0 * tol
    R.check_mx(o.dz, dz, tol)
    mt = (m + 31) // 32 * 32
    assert (o.dz_t.rows, o.dz_t.k, o.dz_t.layout) == (n, mt, layout)
    turned = lambda x: torch.cat([x.t(), x.new_zeros(n, mt - m)], 1)  # noqa: E731
    R.check_mx(o.dz_t, turned(dz), turned(tol))
    close(o.dbias, dz.sum(0), 2.0 ** -16 * dz.abs().sum(0) + tol.sum(0))
    again = F.act_backward(d, z, act, layout=layout, want_dbias=False)
    assert again.dbias is None and torch.equal(again.dz.quantized, o.dz.quantized)


@pytest.mark.parametrize("act", ["relu", "silu", "gelu", "swiglu"])
def test_act_backward_against_differences(F, qlib, act):
    """With one row dbias is dz itself in fp32: against central differences of
    the activation in 64 bits (error of order step^2)."""
    n, step = 256, 1e-4
    z = qlib.make_mxfp8(rand(1, n, seed=95, std=2.0))
    zv = R.value(z)
    d = rand(1, n // 2 if act == "swiglu" else n, seed=96)
    o = F.act_backward(d, z, act)
    for j in (0, 1, 100, 128, 200, 255):
        e = torch.zeros_like(zv)
        e[0, j] = step
        num = (d.to(F64) * (R.act(zv + e, act) - R.act(zv - e, act))).sum() / (2 * step)
        assert abs(float(num) - float(o.dbias[j])) <= 2e-6 * (1 + abs(float(num)) + abs(float(zv[0, j])))


def test_act_backward_special_values(F, qlib):
    """NaN and infinite gradients stay in the blocks that hold them."""
    m, n = 64, 128
    z = qlib.make_mxfp8(rand(m, n, seed=97))
    d = rand(m, n, seed=98)
    clean = F.act_backward(d, z, "gelu")
    d[3, 5], d[40, 70] = float("nan"), float("inf")
    o = F.act_backward(d, z, "gelu")
    q, _ = R.parts(o.dz)
    t, _ = R.parts(o.dz_t)
    assert bool(torch.isnan(q[3, 5])) and bool(torch.isnan(t[5, 3]))
    assert abs(float(q[40, 70])) == 448 and abs(float(t[70, 40])) == 448
    assert int(torch.isnan(q).sum()) == 1 and int(torch.isnan(t).sum()) == 1
    same = torch.ones(m, n, dtype=torch.bool, device=DEV)
    same[3, 0:32], same[40, 64:96] = False, False
    a, b = o.dz.quantized.view(m, n), clean.dz.quantized.view(m, n)
    assert torch.equal(a[same], b[same])
    cols = torch.isfinite(o.dbias)
    assert not bool(cols[5]) and not bool(cols[70]) and int(cols.sum()) == n - 2


@pytest.mark.parametrize("rows,k", [(1, 32), (5, 96), (32, 128), (33, 256), (128, 160),
                                    (300, 4128), (1000, 512)])
@pytest.mark.parametrize("layout", [0, 1, 2])
def test_transpose(F, qlib, rows, k, layout):
    """Every step is exact (values are e4m3 times powers of two), so the codes
    and scales are those of the 64-bit definition."""
    a = qlib.make_mxfp8(rand(rows, k, seed=99, std=5.0), layout)
    out_layout = 1 + rows % 2
    t = F.transpose_mxfp8(a, out_layout)
    rt = (rows + 31) // 32 * 32
    v = torch.cat([R.value(a).t(), torch.zeros(k, rt - rows, dtype=F64, device=DEV)], 1)
    q, sf = R.quantise(v, out_layout)
    assert (t.rows, t.k, t.layout) == (k, rt, out_layout)
    assert torch.equal(t.quantized.view(k, rt), q)
    assert torch.equal(t.block_scales, sf)


@pytest.mark.parametrize("low,high", [(127, 127), (120, 125), (100, 112), (100, 113), (60, 200),
                                      (0, 3), (0, 12), (0, 40), (20, 32), (234, 246)])
@pytest.mark.parametrize("rows,k", [(70, 96), (128, 4128), (40000, 128)])
@pytest.mark.parametrize("kind", ["any", "small", "sparse"])
def test_transpose_scales(F, qlib, low, high, rows, k, kind):
    """Scales of a block that lie near and far from each other, at both ends of
    their range; zeros, columns far below the block's peak, NaN (which a peak
    does not see).  Exact as above."""
    g = torch.Generator(device=DEV).manual_seed(low * 1000 + high + rows)
    q = torch.randint(0, 256, (rows, k), generator=g, device=DEV, dtype=torch.uint8)
    if kind != "any":
        q[q & 0x7f == 0x7f] = 0
    if kind == "small":  # of many columns only the lowest subnormals
        cols = torch.randint(0, 3, (k,), generator=g, device=DEV) > 0
        q = torch.where(cols, q & 0x83, q)
    if kind == "sparse":
        q[torch.rand(rows, k, generator=g, device=DEV) < 0.97] = 0
        q[::3] = 0
    e = torch.randint(low, high + 1, (rows, k // 32), generator=g, device=DEV)
    a = qlib.make_mxfp8(torch.zeros(rows, k, device=DEV), 0)
    a.quantized.copy_(q.view_as(a.quantized))
    a.block_scales.copy_(e.to(torch.uint8).view_as(a.block_scales))
    t = F.transpose_mxfp8(a, 1)
    rt = (rows + 31) // 32 * 32
    v = torch.cat([R.value(a).t(), torch.zeros(k, rt - rows, dtype=F64, device=DEV)], 1)
    bad = v.isnan()
    want, sf = R.quantise(torch.where(bad, torch.zeros_like(v), v), 1)
    assert torch.equal(t.block_scales, sf)
    got = t.quantized.view(k, rt)
    assert bool((got[bad] & 0x7f == 0x7f).all())
    assert torch.equal(got[~bad], want[~bad])


# ------------------------------------------------------------------ long buffers
def test_offsets_past_32_bits(F):
    """More than 2^31 elements: the last rows are those of a short call."""
    rows, k = 70000, 32768
    x = torch.empty(rows, k, dtype=torch.bfloat16, device=DEV)
    x[:-4].fill_(1.0)
    x[-4:] = rand(4, k, seed=101, dtype=torch.bfloat16)
    w = rand(k, seed=102, dtype=torch.bfloat16)
    o = F.rmsnorm_mxfp8(x, w, layout=0)
    s = F.rmsnorm_mxfp8(x[-4:].clone(), w, layout=0)
    assert torch.equal(o.y.quantized.view(rows, k)[-4:], s.y.quantized.view(4, k))
    assert torch.equal(o.y.block_scales[-4 * k // 32:], s.y.block_scales)
    del o
    dx, _ = F.rmsnorm_backward(x, x, torch.ones(rows, device=DEV), w)
    d4, _ = F.rmsnorm_backward(x[-4:].clone(), x[-4:].clone(), torch.ones(4, device=DEV), w)
    assert torch.equal(dx[-4:], d4)
    del dx
    a = F.act_backward(x, None, "none", want_dbias=False)
    last = rows // 32 * 32
    tail = F.act_backward(x[last:].clone(), None, "none", want_dbias=False)
    mt = a.dz_t.k
    assert torch.equal(a.dz.quantized.view(rows, k)[last:], tail.dz.quantized.view(-1, k))
    assert torch.equal(a.dz_t.quantized.view(k, mt)[:, last:], tail.dz_t.quantized.view(k, -1))


# ------------------------------------------------------------------ refusals of the wrappers
def test_wrapper_refusals(F, qlib):
    x, w = rand(4, 256, seed=111), rand(256, seed=112)
    z = qlib.make_mxfp8(x)
    for bad in (lambda: F.rmsnorm_mxfp8(x.half(), w), lambda: F.rmsnorm_mxfp8(x, w, x.bfloat16()),
                lambda: F.rmsnorm_backward(x.bfloat16(), x, w[:4], w),
                lambda: F.rmsnorm_backward(x, x, w[:4].bfloat16(), w),
                lambda: F.gemm_fused(z, z, bias=w[:4].half()), lambda: F.transpose_mxfp8(x),
                lambda: F.act_backward(x, x, "relu"), lambda: F.act_backward(x.half(), z, "relu"),
                lambda: F.rmsnorm_mxfp8("x", w)):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: F.rmsnorm_mxfp8(x, w[:255]), lambda: F.rmsnorm_mxfp8(x, w, x[:3]),
                lambda: F.rmsnorm_mxfp8(x, w, x.cpu()), lambda: F.rmsnorm_mxfp8(x.t(), w[:4]),
                lambda: F.rmsnorm_mxfp8(x[0], w), lambda: F.rmsnorm_backward(x, x, w, w),
                lambda: F.gemm_fused(z, z, bias=w), lambda: F.gemm_fused(z, z, residual=x),
                lambda: F.gemm_fused(z, z, out="fp16"), lambda: F.gemm_fused(z, z, out=x),
                lambda: F.gemm_fused(z, qlib.make_mxfp4(x)), lambda: F.gemm_fused(x, x),
                lambda: F.gemm_fused(z, qlib.make_mxfp8(x, 2)), lambda: F.gemm_fused(z, z, act="x"),
                lambda: F.act_backward(x[:, :32], z, "relu"), lambda: F.act_backward(x, None, "relu"),
                lambda: F.act_backward(x, qlib.make_mxfp8(x), "swiglu")):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: F.rmsnorm_mxfp8(x[:, :40], w[:40]), lambda: F.rmsnorm_mxfp8(x, w, eps=-1),
                lambda: F.rmsnorm_mxfp8(x, w, layout=3), lambda: F.rmsnorm_mxfp8(x[:, 1:33], w[:32]),
                lambda: F.gemm_fused(z, z, out="mxfp8"), lambda: F.gemm_fused(z, z, act="swiglu"),
                lambda: F.transpose_mxfp8(z, 0), lambda: F.act_backward(x, z, "relu", layout=0),
                lambda: F.act_backward(x[:0], None, "none")):
        with pytest.raises(qlib.QGemmError):
            bad()
