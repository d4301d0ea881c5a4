"""Lists of gradients that overlap or name one more than once, and torch's parameters."""
import numpy as np
import pytest
import torch

from novann_amd import optim

pytestmark = pytest.mark.gpu


def test_one_gradient_named_twice_counts_once():
    g = torch.full((3000,), 2.0, device="cuda")
    h = torch.full((16,), 1.0, device="cuda")
    a = np.full(9, 2.0, np.float32)
    n = np.sqrt(4 * 3000 + 16 + 4 * 9)
    lists = [g, h, g, a, g.view(30, 100), a, g[:0], h[:0], a.reshape(3, 3)]
    assert abs(float(optim.grad_norm(lists)) - n) <= 2.0 ** -23 * n
    norm = optim.clip_grad_norm(lists, n / 2, eps=0.0)
    assert abs(float(norm) - n) <= 2.0 ** -23 * n
    assert ((g - 1.0).abs() <= 6 * 2.0 ** -24).all() and ((h - 0.5).abs() <= 6 * 2.0 ** -24).all()
    assert (np.abs(a - 1.0) <= 6 * 2.0 ** -24).all()
    # with outputs, as for a parameter that is named twice: one for each that counts
    outs = [torch.empty(3000, device="cuda"), torch.empty(16, device="cuda")]
    optim.clip_grad_norm([g, g, h], 1e9, out=outs)
    assert torch.equal(outs[0], g) and torch.equal(outs[1], h)
    with pytest.raises(ValueError):
        optim.clip_grad_norm([g, g], 1.0, out=outs)


def test_overlapping_gradients_are_refused():
    buf = torch.ones(100, device="cuda")
    before = buf.clone()
    two = torch.ones(200, device="cuda", dtype=torch.bfloat16)
    for grads, outs in (([buf[:60], buf[40:]], None), ([buf, buf[10:20]], None),
                        ([buf[:50], buf[50:]], [buf[50:], buf[:50]]),
                        ([buf[:40], buf[60:]], [buf[4:44], buf[60:]]),
                        ([buf[:20].clone(), buf[60:80].clone()], [buf[:20], buf[10:30]]),
                        ([two[:100]], [two.view(torch.float32)])):
        with pytest.raises(ValueError):
            optim.clip_grad_norm(grads, 1.0, out=outs)
    assert torch.equal(buf, before)
    # parts of one buffer that do not overlap, and views that are not contiguous, are fine
    optim.clip_grad_norm([buf[:60], buf[60:]], 5.0, eps=0.0)
    m = torch.ones(8, 8, device="cuda")
    norm = optim.clip_grad_norm([m[:, :4], m[:, 4:]], 4.0, eps=0.0)
    assert abs(float(norm) - 8) <= 2.0 ** -20 and ((m - 0.5).abs() <= 6 * 2.0 ** -24).all()
    assert ((buf - 0.5).abs() <= 6 * 2.0 ** -24).all()


def test_torch_parameters_are_clipped_by_their_gradients():
    a = torch.nn.Parameter(torch.ones(5, device="cuda"))
    b = torch.nn.Parameter(torch.ones(4, device="cuda"))
    c = torch.nn.Parameter(torch.ones(3, device="cuda"))
    a.grad, b.grad = torch.full((5,), 2.0, device="cuda"), torch.full((4,), 2.0, device="cuda")
    assert abs(float(optim.grad_norm([a, b, c])) - 6.0) <= 2.0 ** -23 * 6
    optim.clip_grad_norm([a, b, c], 3.0, eps=0.0)
    assert all((p == 1).all() for p in (a, b, c)) and c.grad is None
    for p in (a, b):
        assert ((p.grad - 1.0).abs() <= 6 * 2.0 ** -24).all()
