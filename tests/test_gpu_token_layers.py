"""The token layers' gradients in every form that a caller may hand them."""
import numpy as np
import pytest
import torch

from novann_amd.module import Embedding, LinearCrossEntropy
from tests.token_oracle import cross_entropy_grads, dense, host

pytestmark = pytest.mark.gpu
V, D, N = 90, 32, 50


def tied(dtype):
    np.random.seed(0)
    embed = Embedding(V, D, init=lambda s: np.random.standard_normal(s) / 8, weight_dtype=dtype,
                      factor=2.0, tied=True)
    rng = np.random.default_rng(1)
    t, target = rng.integers(0, V, N), rng.integers(0, V, N)
    target[:3] = -100
    return embed, LinearCrossEntropy(D, V, weight=embed.weight), t, target


def bf16(a):
    return host(torch.from_numpy(np.asarray(a, np.float32)).to(torch.bfloat16))


def check(embed, t, target, h, gx):
    """Both terms in 64 bits, on the operands that the products take (bf16)."""
    w = dense(embed.weight) if embed.weight_dtype else bf16(embed.weight.data)
    hb = bf16(h)
    P, _, want = cross_entropy_grads(hb, w, target, np.full(N, 1 / (N - 3)))
    np.add.at(want, t, 2.0 * np.asarray(gx, np.float64))
    # P rounded to bf16 before its product, fp32 sums
    bound = 2.0 ** -8 * 1.05 * (np.abs(P).T @ np.abs(hb)) + 1e-6
    got = embed.weight.grad
    got = host(got) if isinstance(got, torch.Tensor) else got.astype(np.float64)
    assert (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize("dtype", [None, "e4m3", "e2m1"])
def test_tied_gradients_add_on_arrays(dtype):
    embed, head, t, target = tied(dtype)
    for _ in range(2):  # (a step's gradient replaces the last step's)
        h = embed(t)
        loss = head(h, target)
        gx = head.backward()
        assert isinstance(h, np.ndarray) and isinstance(loss, np.float32)
        assert isinstance(embed.weight.grad, np.ndarray)
        embed.backward(gx)
        assert isinstance(embed.weight.grad, np.ndarray)
        check(embed, t, target, h, gx)


@pytest.mark.parametrize("head_on_device", [False, True])
def test_tied_gradients_add_on_arrays_and_tensors(head_on_device):
    """One of the two layers gets arrays, the other device tensors."""
    embed, head, t, target = tied("e4m3")
    h = embed(t)
    head(torch.from_numpy(h).cuda() if head_on_device else h, target)
    gx = head.backward()
    h = np.asarray(h)
    gx = gx.cpu().numpy() if head_on_device else torch.from_numpy(gx).cuda()
    embed.backward(gx)
    check(embed, t, target, h, gx if head_on_device else gx.cpu().numpy())


def test_tied_gradient_after_zeros():
    """A cleared gradient (zeros, on the host or the device) takes the lookup's own."""
    embed, _, t, _ = tied(None)
    g = np.random.default_rng(2).standard_normal((N, D)).astype(np.float32)
    want, size = np.zeros((V, D)), np.zeros((V, D))
    np.add.at(want, t, 2.0 * g.astype(np.float64))
    np.add.at(size, t, 2.0 * np.abs(g.astype(np.float64)))
    for fresh in (np.zeros((V, D), np.float32), torch.zeros(V, D, device="cuda"), None):
        embed.weight.grad = fresh
        embed(torch.from_numpy(t).cuda())
        embed.backward(torch.from_numpy(g).cuda())
        assert isinstance(embed.weight.grad, torch.Tensor)
        # fp32 sums of at most N terms
        assert (np.abs(host(embed.weight.grad) - want) <= N * 2.0 ** -24 * size).all()
