"""CPU: what the layer operators' binding refuses before it touches a device, shown
with fake tensors (shapes, types and devices without memory)."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode


@pytest.fixture(scope="module")
def F(qlib):
    from cuda_optimazation_b200 import fused
    return fused


def fake(*shape, dtype=torch.float32, device="cuda:0"):
    with FakeTensorMode():
        return torch.empty(*shape, dtype=dtype, device=device)


def held(qlib, rows=128, k=128):
    return qlib.Mxfp8Result(fake(rows * k, dtype=torch.uint8), fake(512, dtype=torch.uint8), rows,
                            k, 1)


def test_status_on_another_device(F, qlib):
    for where in ("cuda:1", "cpu"):
        with pytest.raises(ValueError, match="status"):
            F.gemm_fused(held(qlib), held(qlib),
                         status=fake(1, dtype=torch.int32, device=where))


def test_checkpoint_without_scales(F, qlib):
    z = held(qlib)
    z.block_scales = None
    with pytest.raises(TypeError, match="checkpoint"):
        F.act_backward(fake(128, 128), z, "relu")
    z = held(qlib)
    z.quantized = None
    with pytest.raises(TypeError, match="checkpoint"):
        F.act_backward(fake(128, 128), z, "relu")


class NoTruth:
    def __bool__(self):
        raise RuntimeError("no truth value")


def test_flag_without_a_truth_value(F, qlib):
    with pytest.raises(TypeError, match="truth value"):
        F.gemm_fused(held(qlib), held(qlib), checkpoint=NoTruth())


@pytest.mark.parametrize("layout", [1 + (1 << 32), -(1 << 32), 1 << 40])
def test_layout_beyond_an_int(F, qlib, layout):
    """Not cut down to the layout of its low 32 bits."""
    a = held(qlib)
    for call in (lambda: F.transpose_mxfp8(a, layout),
                 lambda: F.gemm_fused(a, a, out="mxfp8", layout=layout),
                 lambda: F.gemm_fused(a, a, checkpoint=True, checkpoint_layout=layout),
                 lambda: F.act_backward(fake(128, 128), a, "relu", layout=layout),
                 lambda: F.rmsnorm_mxfp8(fake(128, 128), fake(128), layout=layout)):
        with pytest.raises(ValueError, match="layout"):
            call()


@pytest.mark.parametrize("rows,k", [(1 << 31, 1 << 33), (1 << 32, 1 << 32), (1 << 62, 32), (1, 1 << 62)])
def test_shape_whose_size_overflows(F, qlib, rows, k):
    """The buffers' sizes are compared without wrapping round."""
    a = held(qlib)
    a.rows, a.k = rows, k
    b = held(qlib)
    b.k = k
    for call in (lambda: F.transpose_mxfp8(a), lambda: F.gemm_fused(a, a),
                 lambda: F.gemm_fused(b, a)):
        with pytest.raises(ValueError, match="smaller than the shape"):
            call()


class StreamOn:
    """What the operators look at of a torch.cuda.Stream, on a device of its own."""

    def __init__(self, device):
        self.device = torch.device(device)


def test_stream_of_another_device(F, qlib):
    """Not run on the current stream of the operands' device instead."""
    a, x, s = held(qlib), fake(128, 128), StreamOn("cuda:1")
    for call in (lambda: F.rmsnorm_mxfp8(x, fake(128), stream=s),
                 lambda: F.rmsnorm_backward(x, x, fake(128), fake(128), stream=s),
                 lambda: F.gemm_fused(a, a, stream=s),
                 lambda: F.act_backward(x, a, "relu", stream=s),
                 lambda: F.transpose_mxfp8(a, stream=s)):
        with pytest.raises(ValueError, match="stream"):
            call()
