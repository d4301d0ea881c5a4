"""The vocabulary loss's kernel for few tokens (the table read as stored, tokens in
tiles of 32, 64 or 128) with several stages of codes, whole and ragged last rows; and
the products on fp32 hidden states at sizes of large tiles and several pieces."""
import pytest
import torch

from novann_amd import functional as F
from tests import test_gpu_linear_cross_entropy as loss

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N,D,V,wdtype,xdtype", [
    (37, 1024, 5001, "e2m1", "f16"), (100, 640, 3001, "e2m1", "bf16"),
    (128, 2560, 20000, "e2m1", "bf16"), (20, 1056, 30000, "e2m1", "f16"),
    (100, 640, 3001, "bf16", "bf16"), (50, 640, 3001, "f16", "f16"),
    (33, 1000, 2305, "bf16", "bf16"), (1, 1040, 20001, "e4m3", "bf16"),
    (32, 2064, 9999, "e5m2", "f16"), (64, 1040, 4000, "e4m3", "f16"),
    (65, 784, 7777, "e5m2", "bf16")])
def test_several_stages(N, D, V, wdtype, xdtype):
    loss.test_loss(N, D, V, wdtype, xdtype)


@pytest.mark.parametrize("N,D,V,wdtype", [(5000, 700, 33000, "e4m3"), (2048, 512, 20011, "e2m1"),
                                          (1500, 1000, 9001, "f32"), (90, 4096, 18000, "e4m3")])
def test_fp32_hidden_states(N, D, V, wdtype):
    """fp32 x and tables are rounded to bf16 first: what bf16 ones give, unrounded."""
    x, w, w64, t = loss.inputs(N, D, V, wdtype, "f32", seed=12)
    ids = torch.from_numpy(t).cuda()
    xb, wb = x.to(torch.bfloat16), w
    if wdtype == "f32":
        wb = w.data.to(torch.bfloat16)
    value, lse = F.linear_cross_entropy(x, w, ids, extras=True)
    value_b, lse_b = F.linear_cross_entropy(xb, wb, ids, extras=True)
    assert torch.equal(value, value_b) and torch.equal(lse, lse_b)
    gx, gw = F.linear_cross_entropy_backward(x, w, ids, lse)
    assert gx.dtype == torch.float32 and gw.dtype == torch.float32
    gx_b, gw_b = F.linear_cross_entropy_backward(xb, wb, ids, lse, weight_grad_dtype="f32")
    assert torch.equal(gx.to(torch.bfloat16), gx_b) and torch.equal(gw, gw_b)
    assert torch.isfinite(gx).all() and torch.isfinite(gw).all() and gx.any() and gw.any()
