"""The token operators together: the layers, and the example's training steps."""
import os
import sys

import numpy as np
import pytest
import torch

from novann_amd import functional as F
from novann_amd import optim
from novann_amd.module import Embedding, LinearCrossEntropy
from tests.token_oracle import cross_entropy, cross_entropy_grads, dense, host

pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(os.path.dirname(__file__), "..", "examples"))


def small(shape):
    return np.random.standard_normal(shape) / 8


@pytest.mark.parametrize("dtype", [None, "e4m3", "e2m1"])
def test_tied_layers_add_their_gradients(dtype):
    np.random.seed(0)
    V, D, N = 90, 32, 50
    embed = Embedding(V, D, init=small, weight_dtype=dtype, factor=2.0, tied=True)
    head = LinearCrossEntropy(D, V, weight=embed.weight)
    assert head.weight is embed.weight and head.parameters() == []
    rng = np.random.default_rng(1)
    t, target = rng.integers(0, V, N), rng.integers(0, V, N)
    target[:3] = -100
    h = embed(torch.from_numpy(t).cuda())
    loss = head(h, torch.from_numpy(target).cuda())
    gx = head.backward()
    first = embed.weight.grad
    embed.backward(gx)
    assert embed.weight.grad is first
    # the formulas on the operands that the products take (bf16)
    w = dense(embed.weight) if dtype else embed.weight.data.astype(np.float64)
    wb, hb = (host(torch.from_numpy(a.astype(np.float32)).to(torch.bfloat16)) if not dtype or i
              else a for i, a in enumerate((w, host(h))))
    each, _, _ = cross_entropy(hb, wb, target)
    n = N - 3
    assert abs(float(loss) - each.sum() / n) <= 1e-5
    P, want_x, want_w = cross_entropy_grads(hb, wb, target, np.full(N, 1 / n))
    np.add.at(want_w, t, 2.0 * host(gx))
    # P rounded to bf16 before its product, fp32 sums
    bound = 2.0 ** -8 * 1.05 * (np.abs(P).T @ np.abs(hb)) + 1e-6
    assert (np.abs(host(embed.weight.grad) - want_w) <= bound).all()


def test_layers_take_numpy():
    np.random.seed(1)
    V, D = 40, 16
    embed, head = Embedding(V, D, init=small), LinearCrossEntropy(D, V, init=small)
    t = np.arange(8).reshape(2, 4)
    h = embed(t)
    assert isinstance(h, np.ndarray) and h.shape == (2, 4, D)
    loss = head(h.reshape(8, D), np.arange(8))
    g = head.backward()
    assert isinstance(loss, np.float32) and g.shape == (8, D) and g.dtype == np.float32
    embed.backward(g.reshape(2, 4, D))
    assert embed.weight.grad.shape == (V, D) and head.weight.grad.shape == (V, D)
    norm = optim.clip_grad_norm(embed.parameters() + head.parameters(), 1e-3)
    total = sum((p.grad.astype(np.float64) ** 2).sum() for p in (embed.weight, head.weight))
    assert float(norm) > 1e-3 and abs(np.sqrt(total) - 1e-3) < 1e-5
    with pytest.raises(ValueError):
        LinearCrossEntropy(D, V + 1, weight=embed.weight)


@pytest.mark.parametrize("dtype", ["e4m3", "e2m1"])
def test_example_learns(dtype):
    from token_model import train
    losses, norms = train(vocab=500, width=64, batch=2048, steps=80, dtype=dtype)
    # from at least the uniform loss to under half of it (the data's entropy: 1.39)
    assert losses[0] > 0.9 * np.log(500) and np.mean(losses[-5:]) < 0.5 * np.log(500)
    assert np.isfinite(norms).all()


def test_factor_and_dtype():
    np.random.seed(2)
    embed = Embedding(10, 8, init=small, factor=3.0, out_dtype="bf16")
    t = torch.arange(10, device="cuda")
    assert torch.equal(embed(t), F.embedding(t, embed.weight, factor=3.0, out_dtype="bf16"))
