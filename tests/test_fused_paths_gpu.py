"""GPU: the layer operators on the far side of each rule by which they choose a
kernel or a schedule, against their definitions in 64 bits (tolerances as in
test_fused_gpu.py)."""
import pytest
import torch

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
