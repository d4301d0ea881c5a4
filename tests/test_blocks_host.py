"""The shapes that the FP8 blocks' and layer norm's entry points take and give, without a
GPU: tensors lie in host memory and no kernel runs."""
import numpy as np
import pytest
import torch

from novann_amd import functional as F
from novann_amd import quant


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
