"""LayerNorm, BlockLinear and AdamW together, as a model trains and serves with them."""
import os
import sys

import numpy as np
import pytest
import torch

from novann_amd import functional as F
from novann_amd import optim, quant
from novann_amd.module import BlockLinear, LayerNorm
from tests.token_oracle import host

pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(os.path.dirname(__file__), "..", "examples"))


def layers(D, V, **kw):
    np.random.seed(3)
    norm = LayerNorm(D, serve_dtype="e4m3")
    lin = BlockLinear(D, V, init=lambda s: np.random.standard_normal(s) / np.sqrt(D), **kw)
    norm.gamma.data.copy_(1 + 0.1 * torch.randn(D, device="cuda"))
    norm.beta.data.copy_(0.1 * torch.randn(D, device="cuda"))
    if lin.bias is not None:
        lin.bias.data.copy_(torch.randn(1, V, device="cuda"))
    return norm, lin


@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("N,D,V", [(1, 64, 40), (50, 200, 130), (300, 784, 257)])
def test_a_training_step(N, D, V, bias):
    norm, lin = layers(D, V, bias=bias, grad_dtype="e5m2")
    x = torch.randn(N, D, device="cuda").bfloat16()
    g = (torch.randn(N, V, device="cuda") / 8).bfloat16()
    h = norm(x)
    y = lin(h)
    # the layers are the operators
    h2, mean, rstd = F.layer_norm(x, norm.gamma, norm.beta, extras=True)
    assert h.dtype == x.dtype and torch.equal(h, h2)
    assert torch.equal(y, F.block_linear(h, lin.weight, lin.bias))
    gh = lin.backward(g)
    gx = norm.backward(gh)
    gi, gw, gb = F.block_linear_backward(g, h, lin.weight, bias, grad_dtype="e5m2",
                                         weight_grad_dtype="f32")
    assert torch.equal(gh, gi) and torch.equal(lin.weight.grad, gw)
    assert gw.dtype == torch.float32 and (not bias or torch.equal(lin.bias.grad, gb))
    want = F.layer_norm_backward(gi, x, norm.gamma, mean, rstd)
    for a, b in zip((gx, norm.gamma.grad, norm.beta.grad), want):
        assert torch.equal(a, b)
    params = norm.parameters() + lin.parameters()
    assert len(params) == (4 if bias else 3)
    before = lin.weight.master.clone()
    total = optim.clip_grad_norm(params, 0.5)
    assert torch.isfinite(total)
    for kind in ("f32", "8bit"):
        opt = optim.AdamW(params, lr=1e-2, weight_decay=0.1, state_dtype=kind)
        gamma = norm.gamma.data.clone()
        opt.step()
        # (gamma is not decayed: a step of Adam's first length, lr, where its gradient is not 0)
        moved = (norm.gamma.data - gamma).abs()
        assert float(moved.max()) <= 1e-2 * 1.001
    assert not torch.equal(lin.weight.master, before)
    q, t, _ = quant.make_blocks(lin.weight.master, "e4m3", 128, transposed=True)
    assert torch.equal(lin.weight.codes.view(torch.uint8), q.data.view(torch.uint8))
    assert torch.equal(lin.weight.codes_t.view(torch.uint8), t.data.view(torch.uint8))
    opt.zero_grad(set_to_none=True)
    assert lin.weight.grad is None and norm.gamma.grad is None


@pytest.mark.parametrize("N", [1, 5, 40, 200])
def test_serving(N):
    """In eval mode the norm hands over FP8 blocks: the same bits as quantizing its output."""
    norm, lin = layers(300, 130)
    x = torch.randn(N, 300, device="cuda")
    y = lin(norm(x))
    norm.eval(), lin.eval()
    blocks = norm(x)
    assert isinstance(blocks, quant.BlockQuantized) and blocks.dtype == "e4m3"
    assert torch.equal(lin(blocks), y)
    for layer in (norm, lin):
        with pytest.raises(RuntimeError):
            layer.backward(x)
    norm.train(), lin.train()
    assert torch.equal(lin(norm(x)), y)


@pytest.mark.parametrize("shape", [(300,), (2, 20, 300), (3, 1, 4, 300)])
def test_serving_keeps_the_leading_dimensions(shape):
    """The same rows as of the flattened input, in the input's shape."""
    norm, lin = layers(300, 130)
    norm.eval(), lin.eval()
    x = torch.randn(shape, device="cuda")
    y = lin(norm(x))
    assert y.shape == (*shape[:-1], 130)
    assert torch.equal(y.view(-1, 130), lin(norm(x.view(-1, 300))))
    assert norm(x).shape == (x.numel() // 300, 300)


def test_arrays():
    norm, lin = layers(70, 30)
    x = np.random.default_rng(0).standard_normal((6, 70))
    y = lin(norm(x))
    assert isinstance(y, np.ndarray) and y.dtype == np.float32 and y.shape == (6, 30)
    gx = norm.backward(lin.backward(np.ones((6, 30), np.float32)))
    assert isinstance(gx, np.ndarray) and gx.shape == (6, 70)
    opt = optim.AdamW(norm.parameters() + lin.parameters(), lr=0.01)
    opt.step()
    assert np.isfinite(lin(norm(x))).all()


def test_gradient_of_the_chain():
    """The layers' gradients against the 64-bit formulas through the values that the product
    reads: h's blocks, the gradient's, the weight's."""
    N, D, V = 60, 256, 140
    norm, lin = layers(D, V)
    x = torch.randn(N, D, device="cuda")
    g = torch.randn(N, V, device="cuda")
    h = norm(x)
    lin(h)
    gx = norm.backward(lin.backward(g))
    W = host(lin.weight.dequantize())
    G = host(quant.dequantize_blocks(quant.quantize_blocks(g)))
    dh = G @ W
    X = host(x)
    mean = X.mean(1, keepdims=True)
    rstd = 1 / np.sqrt(((X - mean) ** 2).mean(1, keepdims=True) + 1e-5)
    n, s = (X - mean) * rstd, dh * host(norm.gamma.data)
    want = rstd * (s - s.mean(1, keepdims=True) - n * (s * n).mean(1, keepdims=True))
    # the product's sums are off by its 2^-12 of the largest product a block and more; fp32
    # elsewhere
    size = np.abs(G).max(1)[:, None] * np.abs(W).max(0)[None, :] * 2 * 2.0 ** -10
    assert (np.abs(host(gx) - want) <= rstd * (size + size.mean(1, keepdims=True) * 2
                                               * (1 + np.abs(n))) + 1e-5 * np.abs(want).max()).all()


def test_example_runs():
    from token_model import TokenModel, train
    losses, norms = train(vocab=300, width=64, batch=512, steps=5, blocks=True)
    assert np.isfinite(losses).all() and np.isfinite(norms).all() and min(norms) > 0
    np.random.seed(1)
    model = TokenModel(100, 64, "e4m3", blocks=True)
    t = torch.arange(40, device="cuda")
    model.loss(t, t + 1)
    model.backward()
    g = model.head.backward()  # (the same as the one above: it keeps its forward)
    h = model.embed(t)
    y, kept = F.block_linear(model.norm(h), model.mix.weight, model.mix.bias, extras=True)
    gi, gw, gb = F.block_linear_backward(g, kept, model.mix.weight, weight_grad_dtype="f32")
    assert torch.equal(model.mix.weight.grad, gw) and torch.equal(model.mix.bias.grad, gb)
    grads = [model.norm.gamma.grad.clone(), model.norm.beta.grad.clone()]
    model.norm.backward(gi)
    assert torch.equal(grads[0], model.norm.gamma.grad)
    assert torch.equal(grads[1], model.norm.beta.grad)
