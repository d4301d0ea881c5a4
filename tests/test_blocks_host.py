"""The shapes that the FP8 blocks' and layer norm's entry points take and give, without a
GPU: tensors lie in host memory and no kernel runs."""
import numpy as np
import pytest
import torch

from novann_amd import functional as F
from novann_amd import quant
from novann_amd.module import BlockQuantizedParameters


@pytest.fixture
def calls(monkeypatch):
    """The C calls' names, none of which is made."""
    made = []
    monkeypatch.setattr(F, "_device", lambda: torch.device("cpu"))
    monkeypatch.setattr(quant, "on_device", lambda dev, fn, *args: made.append(fn.__name__) or 0)
    return made


@pytest.mark.parametrize("shape", [(40,), (3, 40), (2, 3, 40), (0, 40)])
def test_layer_norm_of_arrays_both_ways(calls, shape):
    """The statistics that the forward gives for an array are the backward's, of one row too."""
    x = np.ones(shape, np.float32)
    y, mean, rstd = F.layer_norm(x, extras=True)
    assert y.shape == shape and mean.shape == rstd.shape == shape[:-1]
    gx, gw, gb = F.layer_norm_backward(x, x, None, mean, rstd)
    assert gx.shape == shape and gw.shape == gb.shape == (40,)
    assert calls == ["novaq_layer_norm", "novaq_layer_norm_backward"]
    with pytest.raises(ValueError):
        F.layer_norm_backward(x, x, None, np.ones(7, np.float32), np.ones(7, np.float32))


@pytest.mark.parametrize("shape", [(40,), (1, 40), (3, 40), (2, 3, 40), (2, 0, 5, 40), (4, 1, 1, 40)])
def test_a_served_chain_keeps_the_leading_dimensions(calls, shape, monkeypatch):
    """layer_norm into blocks and the product behind it: (..., D) to (..., outs)."""
    monkeypatch.setattr(quant, "check_blocks", lambda *a: 0)
    monkeypatch.setattr(F, "_same_device", lambda *a: None)
    w = BlockQuantizedParameters(torch.zeros(30, 128).to(torch.float8_e4m3fn),
                                 torch.zeros(1, 4, dtype=torch.uint8), (30, 40))
    q = F.layer_norm(torch.ones(shape), out_dtype="e4m3")
    assert q.shape == (int(np.prod(shape[:-1])), 40) and q.data.shape == (q.shape[0], 128)
    assert F.block_linear(q, w).shape == (*shape[:-1], 30)
    assert (q.lead is None) == (len(shape) == 2)
    q.lead = (q.shape[0] + 1,)
    with pytest.raises(ValueError):
        F.block_linear(q, w)
