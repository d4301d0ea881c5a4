"""float64 gradients are clipped by a factor of 64 bits."""
import math

import numpy as np
import pytest
import torch

from novann_amd import optim

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("max_norm", [0.75, 1e300])
@pytest.mark.parametrize("inplace", [True, False])
def test_float64_gradients_keep_their_bits(max_norm, inplace):
    """The factor of float64 gradients is a double: 385 squares summed in fp64 (each
    sum at most 2^-53 off, 32 of them behind one another at most), a root, a sum, a
    quotient and a product."""
    rng = np.random.default_rng(0)
    grads = [torch.from_numpy(rng.standard_normal(s)).cuda() for s in ((77, 4), (77,))]
    before = [g.cpu().numpy() for g in grads]
    outs = None if inplace else [torch.empty_like(g) for g in grads]
    eps = 0.1
    norm = optim.clip_grad_norm(grads, max_norm, eps=eps, out=outs)
    n = math.sqrt(math.fsum(float(v) ** 2 for g in before for v in g.ravel()))
    assert abs(float(norm) - n) <= 2.0 ** -23 * n
    coef = min(1.0, max_norm / (n + eps))
    for got, g in zip(outs or grads, before):
        want = g * coef
        assert (np.abs(got.cpu().numpy() - want) <= 40 * 2.0 ** -53 * np.abs(want)).all()


def test_float64_beside_others_beyond_fp32():
    """A norm that fp32 does not hold still scales every gradient by its factor."""
    grads = [torch.full((4,), 1e60, device="cuda", dtype=torch.float64),
             torch.full((3,), 1e30, device="cuda")]
    norm = optim.clip_grad_norm(grads, 1e59, eps=0.0)
    assert float(norm) == np.inf
    assert np.allclose(grads[0].cpu().numpy(), 5e58, rtol=1e-15, atol=0)
    # (the factor rounded to fp32, and a product)
    assert np.allclose(grads[1].cpu().numpy(), 5e28, rtol=2.0 ** -22, atol=0)
