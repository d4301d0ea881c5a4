"""What is not finite stays so through the products of FP8 blocks: an infinity in a layer's
operand becomes a NaN code, whose rows of the product are NaN, and nothing else changes.
(quantize_blocks alone saturates it, as the casts do.)"""
import numpy as np
import pytest
import torch

from novann_amd import functional as F
from novann_amd import optim, quant
from novann_amd.module import BlockQuantizedParameters

pytestmark = pytest.mark.gpu
INF = float("inf")
# one row, the stream kernel's, tiles in both orders apart and together, ragged ones
SHAPES = [(1, 128, 40), (20, 300, 64), (130, 257, 140), (1700, 1100, 130)]


def make(N, D, V, dtype):
    rng = np.random.default_rng(N + D)
    x, g = (torch.from_numpy(rng.standard_normal(s).astype(np.float32)).cuda().to(dtype)
            for s in ((N, D), (N, V)))
    w = BlockQuantizedParameters.from_float(rng.standard_normal((V, D)).astype(np.float32))
    return x, g, w


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N,D,V", SHAPES)
def test_input(N, D, V, dtype, sign, fmt):
    x, g, w = make(N, D, V, dtype)
    r, k = N // 2, D // 3
    x[r, k] = 0
    clean = F.block_linear(x, w, input_dtype=fmt)
    gw = F.block_linear_backward(g, x, w, input_dtype=fmt)[1]
    x[r, k] = sign * INF
    rows, cols = torch.arange(N) != r, torch.arange(D) != k
    y, kept = F.block_linear(x, w, input_dtype=fmt, extras=True)
    for got in (y, F.block_linear(x, w, input_dtype=fmt)):
        assert torch.isnan(got[r]).all() and torch.equal(got[rows], clean[rows])
    for given in (x, kept):
        got = F.block_linear_backward(g, given, w, input_dtype=fmt)[1]
        assert torch.isnan(got[:, k]).all() and torch.equal(got[:, cols], gw[:, cols])


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("N,D,V", SHAPES)
def test_gradient(N, D, V, fmt):
    """An overflowed fp16 gradient shows in every gradient that it has a part in, and so in
    their norm; its neighbours in its blocks are neither clipped nor flushed."""
    x, g, w = make(N, D, V, torch.float16)
    r, n = N // 2, V // 3
    g[r, n] = 0
    clean = F.block_linear_backward(g, x, w, grad_dtype=fmt)
    g[r, n] = INF
    gi, gw, gb = F.block_linear_backward(g, x, w, grad_dtype=fmt)
    rows, outs = torch.arange(N) != r, torch.arange(V) != n
    assert torch.isnan(gi[r]).all() and torch.equal(gi[rows], clean[0][rows])
    assert torch.isnan(gw[n]).all() and torch.equal(gw[outs], clean[1][outs])
    assert gb[0, n] == INF and torch.equal(gb[0, outs], clean[2][0, outs])
    assert not torch.isfinite(optim.grad_norm([gw]))


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("D", [100, 1000, 5000, 17000])
def test_norm(D, fmt):
    """An infinite shift: a NaN code in its column, the others as if it were not there."""
    x = torch.randn(5, D, device="cuda")
    b = torch.randn(D, device="cuda")
    c = D // 2
    b[c] = -INF
    q = F.layer_norm(x, None, b, out_dtype=fmt)
    y = F.layer_norm(x, None, b)
    y[:, c] = 0
    want = quant.quantize_blocks(y, fmt)
    codes = want.data.view(torch.uint8)
    codes[:, c] = 0xFF
    assert torch.equal(q.exponents, want.exponents)
    assert torch.equal(q.data.view(torch.uint8), codes)
    assert torch.isnan(quant.dequantize_blocks(q)[:, c]).all()
