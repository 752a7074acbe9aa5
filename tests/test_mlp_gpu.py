"""GPU: the gated MLP block on the layer operators against the same block in
fp32 with autograd.

Every MXFP8 rounding is off by at most 2^-4 of a value, in the mean square by
2^-4 / sqrt(3) = 3.6 %.  A product of two rounded operands is off by about
sqrt(2) of that (5.1 %); the output has two such products behind each other
(7.2 %, the gate's slope included 9 %), of which the residual takes its share
without error; a gradient has up to five roundings and products in its path
(sqrt(10) x 3.6 % = 11.4 %, with slopes and the double rounding of the turned
operands below 20 %)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mlp(qlib):
    from cuda_optimazation_b200 import mlp
    return mlp


def reference(block, x, residual, dout):
    w = [t.detach().clone().requires_grad_(True)
         for t in (block.norm, block.gate, block.up, block.down)]
    h = (x.float() + (0 if residual is None else residual.float())).requires_grad_(True)
    y = h * (h.square().mean(-1, keepdim=True) + block.eps).rsqrt() * w[0]
    out = (torch.nn.functional.silu(y @ w[1].t()) * (y @ w[2].t())) @ w[3].t() + h
    out.backward(dout.float())
    return out.detach(), h.grad, [t.grad for t in w]


def off(got, ref):
    return float((got.float() - ref).norm() / ref.norm())


@pytest.mark.parametrize("tokens,hidden,inter", [(1, 256, 128), (77, 512, 1408), (300, 1024, 2816)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_block_against_fp32(mlp, tokens, hidden, inter, dt):
    block = mlp.random_block(hidden, inter, seed=3)
    g = torch.Generator(device="cuda").manual_seed(4)
    x, r, d = (torch.randn(tokens, hidden, generator=g, device="cuda").to(dt) for _ in range(3))
    out, saved = block.forward(x, r, train=True)
    ref, dx, dw = reference(block, x, r, d)
    assert out.dtype == dt and off(out, ref) < 0.10
    plain, none = block.forward(x, r)
    assert none is None and torch.equal(plain, out)
    grads = block.backward(d, saved)
    assert grads.x.dtype == dt and off(grads.x, dx) < 0.20
    for got, want in zip((grads.norm, grads.gate, grads.up, grads.down), dw):
        assert got.dtype == torch.float32 and got.shape == want.shape and off(got, want) < 0.20


def test_training_lowers_the_loss(mlp):
    block, target = mlp.random_block(512, 1024, 1), mlp.random_block(512, 1024, 2)
    x = torch.randn(512, 512, generator=torch.Generator(device="cuda").manual_seed(5),
                    device="cuda").to(torch.bfloat16)
    want = target.forward(x)[0].float()
    losses = []
    for _ in range(6):
        out, saved = block.forward(x, train=True)
        err = out.float() - want
        losses.append(float(err.square().mean()))
        block.step(block.backward((err / 512).to(torch.bfloat16), saved), 0.5)
    assert losses[-1] < 0.9 * losses[0] and all(b < a for a, b in zip(losses, losses[1:]))


def test_block_in_a_graph(mlp):
    """The block's calls are stream-ordered and need no host synchronisation: a
    captured forward and backward replays on new contents."""
    block = mlp.random_block(512, 1024, 6)
    x = torch.randn(64, 512, device="cuda").to(torch.bfloat16)
    d = torch.randn(64, 512, device="cuda").to(torch.bfloat16)
    block.backward(d, block.forward(x, train=True)[1])  # warm-up
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, saved = block.forward(x, train=True)
        grads = block.backward(d, saved)
    x.copy_(torch.randn(64, 512, device="cuda"))
    graph.replay()
    want, saved = block.forward(x, train=True)
    assert torch.equal(out, want)
    again = block.backward(d, saved)
    assert torch.equal(grads.x, again.x) and torch.equal(grads.gate, again.gate)


def test_shape_refusals(mlp):
    t = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
    with pytest.raises(ValueError):
        mlp.GatedMlp(t(256), t(128, 256), t(128, 128), t(256, 128))
    with pytest.raises(ValueError):
        mlp.GatedMlp(t(256), t(96, 256), t(96, 256), t(256, 96))  # not whole gate blocks


def test_command(mlp, capsys):
    assert mlp.main(["--tokens", "256", "--hidden", "512", "--inter", "1024", "--steps", "2"]) == 0
    text = capsys.readouterr().out
    assert text.count("loss") == 2 and "one token" in text
