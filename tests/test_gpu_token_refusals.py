"""What the token operators' Python entry points refuse."""
import numpy as np
import pytest
import torch

from novann_amd import functional as F
from novann_amd import optim
from novann_amd.module import Parameters, QuantizedParameters

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def w():
    return QuantizedParameters.from_float(np.ones((20, 16), np.float32), "e4m3")


def test_embedding(w):
    with pytest.raises(ValueError):
        F.embedding(np.array([0, 20]), w)            # host ids are checked
    with pytest.raises(ValueError):
        F.embedding(torch.tensor([-1]), w)           # (a CPU tensor too)
    with pytest.raises(TypeError):
        F.embedding(np.array([0.5]), w)
    with pytest.raises(TypeError):
        F.embedding(torch.zeros(2, device="cuda"), w)
    with pytest.raises(TypeError):
        F.embedding(torch.zeros(2, dtype=torch.bool, device="cuda"), w)
    with pytest.raises(TypeError):
        F.embedding(np.array([1]), w, out_dtype="e4m3")
    with pytest.raises(ValueError):
        F.embedding(np.array([1]), Parameters(np.ones((2, 3, 4), np.float32)))
    short = QuantizedParameters(w.codes[:10], w.shape, w.dtype, w.scale)
    with pytest.raises(ValueError):
        F.embedding(np.array([1]), short)


def test_embedding_backward(w):
    t = torch.zeros(3, dtype=torch.int64, device="cuda")
    g = torch.zeros(3, 16, device="cuda")
    with pytest.raises(ValueError):
        F.embedding_backward(g[:2], t, w)
    with pytest.raises(ValueError):
        F.embedding_backward(g[:, :8], t, w)
    with pytest.raises(ValueError):
        F.embedding_backward(g, t, w, accumulate=True)
    with pytest.raises(ValueError):
        F.embedding_backward(g, t, w, out=torch.zeros(20, 15, device="cuda"))
    with pytest.raises(ValueError):
        F.embedding_backward(g, t, w, out=torch.zeros(16, 20, device="cuda").t())
    with pytest.raises(TypeError):
        F.embedding_backward(g, t, w, out=torch.zeros(20, 16, device="cuda").double())
    with pytest.raises(TypeError):
        F.embedding_backward(g, t, w, out=np.zeros((20, 16), np.float32))
    with pytest.raises(ValueError):
        F.embedding_backward(g, t, w, out=torch.zeros(20 * 16 + 1, device="cuda")[1:].view(20, 16))


def test_linear_cross_entropy(w):
    x = torch.zeros(4, 16, device="cuda", dtype=torch.bfloat16)
    t = torch.zeros(4, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError):
        F.linear_cross_entropy(x[0], w, t)
    with pytest.raises(ValueError):
        F.linear_cross_entropy(x[:, :8], w, t)
    with pytest.raises(ValueError):
        F.linear_cross_entropy(x, w, t[:3])
    with pytest.raises(ValueError):
        F.linear_cross_entropy(x, w, t, reduction="median")
    with pytest.raises(ValueError):
        F.linear_cross_entropy(x, w, np.array([0, 1, 2, 20]))
    with pytest.raises(TypeError):
        F.linear_cross_entropy(x, w, t.float())
    F.linear_cross_entropy(x, w, np.array([0, 1, 2, -100]))
    lse = torch.zeros(4, device="cuda")
    with pytest.raises(ValueError):
        F.linear_cross_entropy_backward(x, w, t, lse[:2])
    with pytest.raises(ValueError):
        F.linear_cross_entropy_backward(x, w, t, lse, grad=torch.ones(4, device="cuda"))
    with pytest.raises(ValueError):
        F.linear_cross_entropy_backward(x, w, t, lse, grad=torch.ones(1, device="cuda"),
                                        reduction="none")
    with pytest.raises(TypeError):
        F.linear_cross_entropy_backward(x, w, t, lse, weight_grad_dtype="e4m3")


def test_clip_grad_norm():
    g = torch.ones(4, device="cuda")
    with pytest.raises(TypeError):
        optim.clip_grad_norm([g.int()], 1.0)
    with pytest.raises(ValueError):
        optim.clip_grad_norm([g.cpu()], 1.0)
    with pytest.raises(ValueError):
        optim.clip_grad_norm([g], -1.0)
    with pytest.raises(ValueError):
        optim.clip_grad_norm([g], 1.0, eps=float("nan"))
    with pytest.raises(ValueError):
        optim.clip_grad_norm([g], 1.0, out=[])
    with pytest.raises(ValueError):
        optim.clip_grad_norm([g], 1.0, out=[torch.empty(3, device="cuda")])
    with pytest.raises(ValueError):
        optim.clip_grad_norm([g], 1.0, out=[torch.empty(4)])
    with pytest.raises(TypeError):
        optim.clip_grad_norm([np.ones(3, np.int64)], 1.0)
