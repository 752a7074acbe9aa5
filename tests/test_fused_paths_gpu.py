"""GPU: the layer operators on the far side of each rule by which they choose a
kernel or a schedule, against their definitions in 64 bits (tolerances as in
test_fused_gpu.py)."""
import pytest
import torch

import fused_ref as R
import test_fused_gpu as base
from test_fused_gpu import gemm_case

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")


@pytest.fixture(scope="module")
def F(qlib):
    from cuda_optimazation_b200 import fused
    return fused


# ------------------------------------------------------------------ GEMM of few rows
@pytest.mark.parametrize("blocks", [1, 2, 4, 6, 8, 10, 12, 14, 16])
@pytest.mark.parametrize("m", [1, 9, 17, 65, 128])
def test_few_rows_cluster_sizes(F, qlib, m, blocks):
    """Clusters of 1 to 8 CTAs (half the 128-byte K blocks); rows that leave some
    warps, or the second of a warp's two rows, without one; a last tile of which
    most columns lie beyond the matrix."""
    gemm_case(F, qlib, m, 204, blocks * 128, act="silu", bias="f32", res="bf16",
              out="bf16" if m % 2 else "f32")
    gemm_case(F, qlib, m, 160, blocks * 128, act="none", out="mxfp8", ckpt=True)


@pytest.mark.parametrize("m,n,k,act", [
    (1, 28672, 1280, "swiglu"),   # 112 tiles: two CTAs an SM in clusters of two
    (1, 16384, 2304, "swiglu"),   # 64 tiles: more CTAs to a cluster
    (16, 12800, 1280, "none"),    # the same, ungated
    (64, 12800, 4224, "none"),    # 64 rows: from 33 blocks on
    (3, 28672, 1280, "none"),     # more tiles than SMs
    (5, 40064, 96, "silu"),       # more than twice as many
])
@pytest.mark.parametrize("fmt", ["mxfp8", "nvfp4"])
def test_few_rows_two_ctas_an_sm(F, qlib, m, n, k, act, fmt):
    k = 2 * k if fmt == "nvfp4" else k  # the same number of 128-byte blocks
    gemm_case(F, qlib, m, n, k, fmt, act=act, out="mxfp8", ckpt=m == 1)
    gemm_case(F, qlib, m, n, k, fmt, act=act, bias="bf16", res="f32", out="bf16")


# ------------------------------------------------------------------ GEMM of many rows
def pair_case(F, qlib, m, n, k, fmt, act, out, bias, res, ckpt, pad):
    """gemm_case with rows of the residual and of a given output `pad` further apart
    (0: on 16 bytes, the epilogues that hold a row), and the call once more."""
    a, av = base.operand(qlib, m, k, fmt, 131)
    b, bv = base.operand(qlib, n, k, fmt, 132, k ** -0.5)
    cols = n // 2 if act == "swiglu" else n
    bt = base.rand(n, seed=133, dtype=base.TYPES[bias]) if bias else None
    rt = base.rand(m, cols, seed=134, std=2.0, dtype=base.TYPES[res], pad=pad) if res else None
    status = torch.zeros(1, dtype=torch.int32, device=DEV)

    def call():
        to = out
        if out != "mxfp8":
            to = torch.full((m, cols + pad), 7.0, dtype=base.TYPES[out], device=DEV)[:, :cols]
        o = F.gemm_fused(a, b, bias=bt, act=act, residual=rt, out=to, checkpoint=ckpt,
                         status=status)
        if out != "mxfp8" and pad:
            assert bool((to._base[:, cols:] == 7.0).all()), "columns beyond the output"
        return o

    o = call()
    assert qlib.read_status(status)[0] == qlib.OK
    z = av @ bv.t()
    tol = 2.0 ** -16 * (av.abs() @ bv.abs().t())
    if bias:
        z, tol = z + bt.double(), tol + 2.0 ** -22 * bt.double().abs()
    y, ty = R.act(z, act), R.act_tol(z, tol, act)
    if res:
        y, ty = y + rt.double(), ty + 2.0 ** -22 * rt.double().abs()
    again = call()
    if out == "mxfp8":
        R.check_mx(o.out, y, ty)
        assert torch.equal(o.out.quantized, again.out.quantized)
        assert torch.equal(o.out.block_scales, again.out.block_scales)
    else:
        base.close(o.out, y, ty + 1.01 * base.STEP[o.out.dtype] * y.abs())
        assert torch.equal(o.out, again.out)
    if ckpt:
        R.check_mx(o.checkpoint, z, tol)
        assert torch.equal(o.checkpoint.quantized, again.checkpoint.quantized)
        assert torch.equal(o.checkpoint.block_scales, again.checkpoint.block_scales)


# 240 tiles of 256 x 256 for 74 pairs: every pair takes several, with the shortest main
# loop (one K block), so that an epilogue meets the next tile's.
@pytest.mark.parametrize("act,out,bias,res,ckpt,pad", [
    ("swiglu", "mxfp8", None, None, True, 0),
    ("swiglu", "mxfp8", "bf16", "bf16", True, 0),
    ("swiglu", "bf16", "f32", "f32", True, 0),
    ("swiglu", "f32", None, "bf16", False, 0),
    ("gelu", "bf16", "bf16", "bf16", False, 0),
    ("gelu", "f32", "f32", "f32", True, 0),
    ("relu", "mxfp8", None, "f32", True, 0),
    ("none", "mxfp8", "f32", None, False, 0),
    ("gelu", "bf16", "bf16", "bf16", True, 3),
    ("silu", "f32", "f32", "f32", False, 3),
    ("none", "mxfp8", None, "bf16", True, 3),
    ("swiglu", "bf16", "bf16", "f32", True, 3),
    ("swiglu", "mxfp8", None, "bf16", True, 3),
    ("swiglu", "f32", None, None, False, 3),
])
@pytest.mark.parametrize("fmt,k", [("mxfp8", 96), ("nvfp4", 192), ("mxfp4", 192)])
def test_pair_several_tiles(F, qlib, act, out, bias, res, ckpt, pad, fmt, k):
    pair_case(F, qlib, 3001, 5120, k, fmt, act, out, bias, res, ckpt, pad)


@pytest.mark.parametrize("m,n", [(3001, 5121), (2999, 5127), (20000, 67)])
@pytest.mark.parametrize("out,res", [("bf16", "f32"), ("f32", "bf16"), ("bf16", None)])
def test_pair_several_odd_tiles(F, qlib, m, n, out, res):
    pair_case(F, qlib, m, n, 160, "mxfp8", "gelu", out, "f32", res, False, 0)


@pytest.mark.parametrize("act,out", [("swiglu", "mxfp8"), ("silu", "bf16"), ("none", "f32")])
def test_pair_long_main_loop(F, qlib, act, out):
    """Several tiles a pair with a main loop longer than the epilogue."""
    pair_case(F, qlib, 2100, 4864, 1024, "mxfp8", act, out, "bf16", "bf16", out == "mxfp8", 0)


def test_gemm_offsets_past_32_bits(F, qlib):
    """More than 2^31 outputs: the last rows are those of a call on them alone."""
    m, n, k, tail = 66000, 32768, 32, 464  # a whole number of row tiles before the tail
    a, _ = base.operand(qlib, m, k, "mxfp8", 141, layout=2)
    b, _ = base.operand(qlib, n, k, "mxfp8", 142, layout=2)
    assert (m - tail) % 256 == 0
    last = qlib.make_mxfp8(base.rand(m, k, seed=141)[-tail:].contiguous(), 2)
    c = torch.zeros(m, n, dtype=torch.bfloat16, device=DEV)
    c[-tail:] = base.rand(tail, n, seed=143, dtype=torch.bfloat16)
    small = c[-tail:].clone()
    o = F.gemm_fused(a, b, residual=c, out=c, checkpoint=True, checkpoint_layout=0)
    s = F.gemm_fused(last, b, residual=small, out=small, checkpoint=True, checkpoint_layout=0)
    assert torch.equal(c[-tail:], small)
    assert torch.equal(o.checkpoint.quantized.view(m, n)[-tail:], s.checkpoint.quantized.view(-1, n))
    assert torch.equal(o.checkpoint.block_scales.view(m, -1)[-tail:],
                       s.checkpoint.block_scales.view(tail, -1))


# ------------------------------------------------------------------ activation backward
# Many tiles: row groups one after the other; every layout of the
# checkpoint, ragged last rows and columns, dbias through the partial sums.
@pytest.mark.parametrize("m", [2500, 2501, 2531])
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu"])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_act_backward_many_tiles(F, qlib, m, act, dt):
    base.test_act_backward(F, qlib, m, 4128, act, dt)


@pytest.mark.parametrize("m,n", [(3001, 8192), (3002, 8448), (4993, 4096)])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_gated_backward_many_tiles(F, qlib, m, n, dt):
    base.test_act_backward(F, qlib, m, n, "swiglu", dt)


# One round of tiles (148 SMs) and one more; dbias of up to 8 row tiles joined in a
# cluster where all clusters find a place, else through the partial sums; (1000, 2048):
# joined in the gated form, not in the ungated one.
@pytest.mark.parametrize("m,n", [(500, 512), (769, 256), (1000, 512), (1024, 256), (1025, 256),
                                 (2000, 256), (9000, 512), (1000, 9728), (1000, 2048),
                                 (500, 4736), (500, 4864), (400, 4096), (900, 1792), (250, 18944),
                                 (250, 19456), (18900, 256)])
@pytest.mark.parametrize("act", ["gelu", "swiglu"])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_act_backward_row_tiles(F, qlib, m, n, act, dt):
    base.test_act_backward(F, qlib, m, n, act, dt)


# ------------------------------------------------------------------ transposition
@pytest.mark.parametrize("rows,k", [(2500, 4128), (10001, 1056), (128, 75808), (75777, 128),
                                    (9473, 1152), (4700, 1024), (4740, 1024)])
@pytest.mark.parametrize("layout", [0, 1, 2])
def test_transpose_many_tiles(F, qlib, rows, k, layout):
    base.test_transpose(F, qlib, rows, k, layout)


@pytest.mark.parametrize("kind", ["any", "small", "sparse"])
@pytest.mark.parametrize("low,high", [(127, 127), (100, 113), (60, 200), (0, 40), (234, 246)])
def test_transpose_scales_many_tiles(F, qlib, low, high, kind):
    base.test_transpose_scales(F, qlib, low, high, 2533, 4128, kind)


def test_transpose_offsets_past_32_bits(F, qlib):
    """More than 2^31 values: the last rows are those of a call on them alone."""
    rows, k, tail = 66048, 32768, 512
    g = torch.Generator(device=DEV).manual_seed(151)
    q = torch.zeros(rows, k, dtype=torch.uint8, device=DEV)
    q[-tail:] = torch.randint(0, 0x7f, (tail, k), generator=g, device=DEV, dtype=torch.uint8)
    e = torch.randint(100, 140, (rows, k // 32), generator=g, device=DEV, dtype=torch.uint8)
    t = F.transpose_mxfp8(qlib.Mxfp8Result(q.view(-1), e.view(-1), rows, k, 0), 2)
    s = F.transpose_mxfp8(qlib.Mxfp8Result(q[-tail:].reshape(-1), e[-tail:].reshape(-1), tail, k, 0),
                          2)
    assert torch.equal(t.quantized.view(k, rows)[:, -tail:], s.quantized.view(k, tail))
    # K-major chunks: a row block's last tail / 128 chunks.
    whole = t.block_scales.view(k // 128, rows // 128, 512)
    assert torch.equal(whole[:, -tail // 128:], s.block_scales.view(k // 128, tail // 128, 512))


# ------------------------------------------------------------------ norm
# Both sides of the rule for the ring: short rows, eight to a CTA, by their bytes and
# their number, and long ones by both or by k alone.
@pytest.mark.parametrize("rows,k", [(6143, 64), (6145, 64), (8200, 128), (8200, 256), (16500, 512),
                                    (16500, 1024), (9000, 32), (8100, 4096), (8200, 4096),
                                    (2040, 8192), (2050, 8192), (301, 16384), (300, 12320)])
@pytest.mark.parametrize("xt,wt", [("bf16", "bf16"), ("f32", "f32"), ("bf16", "f32")])
def test_norm_paths(F, rows, k, xt, wt):
    base.test_norm(F, rows, k, xt, wt)


@pytest.mark.parametrize("rows,k", [(8193, 128), (8193, 256), (16500, 512), (16500, 1024),
                                    (8200, 4096)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_norm_paths_without_a_residual(F, rows, k, dt):
    x, w = base.rand(rows, k, seed=161, dtype=dt), base.rand(k, seed=162, dtype=dt)
    o = F.rmsnorm_mxfp8(x, w, eps=1e-5, layout=k // 128 % 3)
    _, rstd, y = R.norm(x, None, w, 1e-5)
    assert o.h is x
    base.close(o.rstd, rstd, 2.0 ** -16 * rstd)
    R.check_mx(o.y, y, 2.0 ** -15 * y.abs())


# ------------------------------------------------------------------ norm gradient
# Up to 512 rows by columns, or (long bf16 rows) through the ring; beyond by type, width
# and number of rows through the ring or partial sums.
@pytest.mark.parametrize("rows,k", [(512, 64), (513, 64), (290, 16384), (300, 16384), (512, 16416),
                                    (200, 32768), (512, 32768), (513, 32768), (600, 16416),
                                    (512, 9376), (513, 9376), (520, 6144), (600, 12288),
                                    (2367, 256), (2368, 256), (2400, 768), (2400, 800),
                                    (2559, 1024), (2560, 1280), (1300, 1536), (900, 2048),
                                    (1500, 2048), (640, 3104), (900, 4128), (700, 7200)])
@pytest.mark.parametrize("xt,wt", [("bf16", "bf16"), ("f32", "f32"), ("bf16", "f32")])
def test_norm_backward_rows(F, rows, k, xt, wt):
    base.test_norm_backward(F, rows, k, xt, wt)
