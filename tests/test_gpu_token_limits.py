"""Calls whose work needs more threads than one launch may have."""
import numpy as np
import pytest
import torch

from novann_amd import functional as F
from tests.token_oracle import cross_entropy, floats, host

pytestmark = pytest.mark.gpu


def test_loss_of_more_logits_than_one_launch():
    """2^39 logits: their tiles' threads are 2^32."""
    N, D, V = (1 << 22) + 3, 8, (1 << 17) + 1
    rng = np.random.default_rng(0)
    w = floats(rng, (V, D), "bf16", 0.5)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    x = torch.randn(N, D, generator=gen, device="cuda").to(torch.bfloat16)
    ids = torch.randint(0, V, (N,), generator=gen, device="cuda")
    ids[-1], ids[5] = V - 1, -100
    each, lse = F.linear_cross_entropy(x, w, ids, reduction="none", extras=True)
    assert torch.isfinite(each).all() and torch.isfinite(lse).all()
    at = torch.cat([torch.arange(8), torch.from_numpy(rng.integers(0, N, 40)), torch.arange(N - 8, N)])
    x64, w64, t = host(x[at.cuda()]), host(w), ids[at.cuda()].cpu().numpy()
    want, want_lse, _ = cross_entropy(x64, w64, t)
    # fp32 sums of D products, exp, log and the change of base (2^-20)
    e = np.sqrt(D) * 2.0 ** -23 * (np.abs(x64) @ np.abs(w64).T).max() + \
        2.0 ** -20 * (1 + np.abs(want_lse).max())
    assert np.abs(host(lse)[at] - want_lse).max() <= e
    assert np.abs(host(each)[at] - want).max() <= 2 * e
    del x, each, lse
    torch.cuda.empty_cache()


def test_embedding_gradient_of_more_tokens_than_one_launch():
    """Sums of 2^27 tokens join 2^23 parts, 512 threads each; gradients of 0 and 1, whose
    sums fp32 holds exactly in any order."""
    N, V = (1 << 27) + 5, 700
    gen = torch.Generator(device="cuda")
    gen.manual_seed(2)
    ids = torch.randint(0, V, (N,), generator=gen, device="cuda", dtype=torch.int32)
    ids[-3:] = V - 1
    g = torch.randint(0, 2, (N, 1), generator=gen, device="cuda").to(torch.bfloat16)
    got = F.embedding_backward(g, ids, (V, 1))
    want = torch.zeros(V, dtype=torch.float64, device="cuda")
    for k in range(0, N, 1 << 24):
        want += torch.bincount(ids[k:k + (1 << 24)], g[k:k + (1 << 24), 0].double(), V)
    assert torch.equal(got[:, 0].double(), want)
    del ids, g
    torch.cuda.empty_cache()
