"""CPU: an output over one of its inputs with another stride or type, where elements
would not lie on their own, is refused before any CUDA call."""
import pytest

from test_fused_cpu import A, gemm, norm, norm_bwd

B, C = 2 * A, 3 * A


@pytest.mark.parametrize("over", [dict(h=B, x=B, ldx=256, ldh=512, res=C),
                                  dict(h=C, res=C, ldr=512, ldh=256, x=B),
                                  dict(h=C, res=C, ldr=256, ldh=264, x=B, rows=2)])
def test_norm_sum_over_an_input(qlib, over):
    assert norm(qlib.lib(), **over) == qlib.ERR_ARG


def test_norm_gradient_over_dres(qlib):
    assert norm_bwd(qlib.lib(), dx=B, dres=B, lddres=512, lddx=256) == qlib.ERR_ARG


@pytest.mark.parametrize("other", [dict(ldr=512), dict(residual_dtype=0), dict(out_dtype=0),
                                   dict(out_dtype=2, out_sf=A), dict(m=1, residual_dtype=0)])
def test_gemm_over_its_residual(qlib, other):
    assert gemm(qlib, **(dict(residual=A, residual_dtype=1, ldr=256) | other)) == qlib.ERR_ARG
