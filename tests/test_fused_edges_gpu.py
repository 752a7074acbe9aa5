"""GPU: infinities, NaN and zeros where the layer operators' definitions have an
edge, and the errors that a call raises."""
import pytest
import torch

import fused_ref as R

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
INF, NAN = float("inf"), float("nan")


@pytest.fixture(scope="module")
def F(qlib):
    from cuda_optimazation_b200 import fused
    return fused


@pytest.mark.parametrize("m", [1, 70, 20000])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_relu_slope_at_its_edges(F, qlib, m, dt):
    """dz = dout where z > 0 and 0 where z <= 0, whatever dout holds there; a NaN z
    gives NaN.  (m: one tile, few tiles, and enough that row groups come in turn.)"""
    n = 512
    zv = torch.ones(m, n, device=DEV)
    zv[:, 1::4], zv[:, 2::4] = -1.0, 0.0
    z = qlib.make_mxfp8(zv)
    z.quantized.view(m, n)[:, 31] = 0x7f  # column 31 would be 0
    d = torch.full((m, n), 2.0, device=DEV, dtype=dt)
    # In blocks of their own (of rows and columns) where z > 0.
    special = {4: INF, 5: INF, 6: -INF, 9: NAN, 10: NAN, 13: -INF}
    for c, v in special.items():
        d[0, c] = v
    o = F.act_backward(d, z, "relu")
    want = torch.where(zv > 0, d.double(), torch.zeros((), dtype=torch.float64, device=DEV))
    want[:, 31] = NAN
    q, _ = R.parts(o.dz)
    t, _ = R.parts(o.dz_t)
    for got in (q, t[:, :m].t()):
        assert torch.equal(got.isnan(), want.isnan())
        assert bool((got[want == 0] == 0).all())  # (beside an infinity 2 goes to 0 as well)
        assert torch.equal(got.abs() == 448, want.isinf())
    ok = torch.ones(n, dtype=torch.bool, device=DEV)
    ok[31] = ok[4] = False
    assert torch.equal(o.dbias[ok].double(), want[:, ok].sum(0))
    assert bool(o.dbias[31].isnan()) and float(o.dbias[4]) == INF


def test_out_of_memory_error(F, qlib):
    """An output that does not fit raises torch's own error, as torch.empty does."""
    d = torch.zeros(1, 1 << 18, device=DEV, dtype=torch.bfloat16).expand(1 << 21, 1 << 18)
    with pytest.raises(torch.OutOfMemoryError):
        F.act_backward(d, None, "none")
    a = torch.zeros(1, 32768, device=DEV).expand(1 << 25, 32768)
    with pytest.raises(torch.OutOfMemoryError):
        F.rmsnorm_mxfp8(a, a[0])
