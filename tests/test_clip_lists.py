"""Which of the gradients that a list names are clipped (host side, no GPU)."""
import numpy as np
import torch

from novann_amd import optim
from novann_amd.module import Parameters


def same(got, want):
    got, at = got
    assert at is None or at == [g.data_ptr() for g in want]
    return len(got) == len(want) and all(a is b for a, b in zip(got, want))


def test_one_gradient_named_twice_is_taken_once():
    g, h = torch.ones(6), torch.ones(6)
    assert same(optim._gradients([g, h]), [g, h])
    assert same(optim._gradients([g, h, g]), [g, h])
    assert same(optim._gradients([g, g.view(2, 3), h]), [g, h])
    a = np.ones(6, np.float32)
    assert same(optim._gradients([a, g, a, a.reshape(2, 3), g]), [a, g])
    p, q = Parameters(np.zeros(6, np.float32)), Parameters(np.zeros(6, np.float32))
    p.grad = q.grad = g
    assert same(optim._gradients([p, q, p, h, g]), [g, h])
    p.grad = None
    assert same(optim._gradients(iter([p, q])), [g])


def test_other_views_are_other_gradients():
    m = torch.arange(12.0).view(3, 4)
    for pair in ([m[:, :2], m[:, 2:]], [m, m.t()], [m[:, 0], m[:, :1]], [m[:2], m],
                 [m.view(-1)[:6], m.view(-1)[::2]], [m, m.view(torch.int32)]):
        assert same(optim._gradients(pair), pair)
    a = m.numpy()
    for pair in ([a[:, :2], a[:, 2:]], [a, a.T], [a[:2], a]):
        assert same(optim._gradients(pair), pair)
    empty = [m[:0], m[:0], torch.empty(0), torch.empty(0)]
    assert same(optim._gradients(empty), empty)
    assert same(optim._gradients([]), [])


def test_torch_parameters_stand_for_their_gradients():
    a, b, c = (torch.nn.Parameter(torch.ones(3)) for _ in range(3))
    a.grad = torch.full((3,), 2.0)
    c.grad = a.grad
    h = torch.ones(5)
    assert same(optim._gradients([a, b, c]), [a.grad])
    assert same(optim._gradients([h, a]), [h, a.grad])
    assert same(optim._gradients([b]), [])
