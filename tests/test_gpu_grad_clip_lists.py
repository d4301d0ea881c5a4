"""Lists of gradients that overlap, or name one more than once."""
import pytest
import torch

from novann_amd import optim

pytestmark = pytest.mark.gpu


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
