"""Layer norm and its gradients against the formulas in 64 bits, and its FP8 blocks
against those of its fp32 output."""
import numpy as np
import pytest
import torch

from novann_amd import functional as F
from novann_amd import quant
from novann_amd.module import Parameters
from tests.token_oracle import HALF_MIN, HALF_ULP, TORCH, host

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # half a unit of fp32
# one element, below and past each number of threads a row, odd widths, walked rows
WIDTHS = [1, 3, 64, 130, 512, 520, 784, 1024, 1031, 2048, 2056, 4096, 4097, 8192, 8200, 16384,
          16392, 20001]


def data(rng, R, D, dtype):
    x = rng.standard_normal((R, D)) * 2.0 ** rng.integers(-3, 4, (R, 1)) + rng.standard_normal((R, 1))
    t = torch.from_numpy(x.astype(np.float32)).cuda().to(TORCH[dtype])
    w = torch.from_numpy((1 + 0.3 * rng.standard_normal(D)).astype(np.float32)).cuda()
    b = torch.from_numpy((0.3 * rng.standard_normal(D)).astype(np.float32)).cuda()
    return t, w, b


def exact(x, w, b, eps):
    mean = x.mean(-1, keepdims=True)
    c = x - mean
    rstd = 1 / np.sqrt((c * c).mean(-1, keepdims=True) + eps)
    return c * rstd * w + b, c * rstd, mean, rstd


def tolerance(x, w, n, mean, rstd):
    """Of y in fp32: a mean of D sums in chains of at most 16 + 16 and trees is off by 40 U of
    the mean magnitude, which the deviation takes over, with its own rounding; rstd is off
    by 40 U (its sum), 4 more roundings; the product and sum round 4 times."""
    size = np.abs(x).mean(-1, keepdims=True)
    return U * ((42 * size + np.abs(x) + np.abs(mean)) * rstd * np.abs(w) + 50 * np.abs(n * w) + 4)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("D", WIDTHS)
def test_forward(D, dtype):
    rng = np.random.default_rng(D)
    R = 9 if D > 1100 else 70
    x, w, b = data(rng, R, D, dtype)
    y, n, mean, rstd = exact(host(x), host(w), host(b), 1e-5)
    tol = tolerance(host(x), host(w), n, mean, rstd)
    got, gm, gr = F.layer_norm(x, w, b, out_dtype="f32", extras=True)
    assert (np.abs(host(got) - y) <= tol).all()
    assert (np.abs(host(gm) - mean[:, 0]) <= 42 * U * np.abs(host(x)).mean(1)).all()
    size = np.abs(host(x)).mean(1)
    assert (np.abs(host(gr) / rstd[:, 0] - 1) <= 50 * U + 200 * U * size * rstd[:, 0]).all()
    own = F.layer_norm(x, w, b)
    assert own.dtype == x.dtype and torch.equal(own, got.to(x.dtype))
    assert torch.equal(F.layer_norm(x, w, b, out_dtype="bf16"), got.bfloat16())
    assert torch.equal(F.layer_norm(x, out_dtype="f32"),
                       F.layer_norm(x, torch.ones(D), torch.zeros(D), out_dtype="f32"))


@pytest.mark.parametrize("dtype", ["e4m3", "e5m2"])
@pytest.mark.parametrize("D", WIDTHS)
def test_blocks(D, dtype):
    """Blocks of y as quantize_blocks makes them of the fp32 output, bit for bit."""
    rng = np.random.default_rng(D)
    x, w, b = data(rng, 6, D, "bf16")
    x[2] = 1.0             # a constant row: y is the shift
    x[4, D // 2] = float("nan")
    q, mean, rstd = F.layer_norm(x, w, b, out_dtype=dtype, extras=True)
    want = quant.quantize_blocks(F.layer_norm(x, w, b, out_dtype="f32"), dtype)
    assert q.shape == (6, D) and q.dtype == dtype
    assert torch.equal(q.data.view(torch.uint8), want.data.view(torch.uint8))
    assert torch.equal(q.exponents, want.exponents)


@pytest.mark.parametrize("gdt,dtype", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"),
                                       ("f32", "bf16"), ("bf16", "f16")])
@pytest.mark.parametrize("D", WIDTHS)
def test_backward(D, gdt, dtype):
    rng = np.random.default_rng(D + 1)
    R = 13 if D > 1100 else 77
    x, w, b = data(rng, R, D, dtype)
    g = torch.from_numpy(rng.standard_normal((R, D)).astype(np.float32)).cuda().to(TORCH[gdt])
    _, mean, rstd = F.layer_norm(x, w, b, extras=True)
    gx, gw, gb = F.layer_norm_backward(g, x, w, mean, rstd)
    assert gx.dtype == x.dtype and gw.dtype == gb.dtype == torch.float32
    # the formulas, from the statistics that the call was given
    X, G, W, m, r = host(x), host(g), host(w), host(mean)[:, None], host(rstd)[:, None]
    n, h = (X - m) * r, G * W
    want = r * (h - h.mean(1, keepdims=True) - n * (h * n).mean(1, keepdims=True))
    # n is off by 3 U; the means of D by 42 U of their terms' mean size; 8 roundings
    size = np.abs(h).mean(1, keepdims=True) + np.abs(n) * np.abs(h * n).mean(1, keepdims=True)
    tol = U * r * (8 * np.abs(h) + 60 * size + 3 * (np.abs(X) + np.abs(m)) * r * np.abs(
        (h * n).mean(1, keepdims=True)))
    tol += HALF_ULP[dtype] * (np.abs(want) + tol) + HALF_MIN[dtype]
    assert (np.abs(host(gx) - want) <= tol).all()
    # sums of R terms: at most R roundings, 4 in a term
    assert (np.abs(host(gw) - (G * n).sum(0)) <=
            (R + 8) * U * (np.abs(G) * (np.abs(X) + np.abs(m)) * r).sum(0)).all()
    assert (np.abs(host(gb) - G.sum(0)) <= (R + 4) * U * np.abs(G).sum(0)).all()
    again = F.layer_norm_backward(g, x, w, mean, rstd)
    assert all(torch.equal(a, c) for a, c in zip(again, (gx, gw, gb)))


def test_gradients_by_differences():
    rng = np.random.default_rng(5)
    x, w, b = data(rng, 4, 50, "f32")
    g = rng.standard_normal((4, 50))
    _, mean, rstd = F.layer_norm(x, w, b, extras=True)
    gx, gw, gb = (host(t) for t in F.layer_norm_backward(
        torch.from_numpy(g.astype(np.float32)).cuda(), x, w, mean, rstd))
    X, W, B, eps = host(x), host(w), host(b), 1e-6

    def loss(X, W, B):
        return (exact(X, W, B, 1e-5)[0] * g).sum()

    for a, grad in ((X, gx), (W, gw), (B, gb)):
        for i in [0, a.size // 2, a.size - 1]:
            keep = a.reshape(-1)[i]
            a.reshape(-1)[i] = keep + eps
            up = loss(X, W, B)
            a.reshape(-1)[i] = keep - eps
            down = loss(X, W, B)
            a.reshape(-1)[i] = keep
            # second differences are of the order eps^2, roundings of fp32 of the terms'
            assert abs((up - down) / (2 * eps) - grad.reshape(-1)[i]) <= 1e-4 * (
                1 + abs(grad.reshape(-1)[i]))


def test_many_rows():
    """More rows than workgroups take at once, an odd number."""
    rng = np.random.default_rng(6)
    for R, D in ((5003, 136), (2601, 1500)):
        x, w, b = data(rng, R, D, "bf16")
        g = torch.randn(R, D, device="cuda").bfloat16()
        y, mean, rstd = F.layer_norm(x, w, b, out_dtype="f32", extras=True)
        want, n, m, r = exact(host(x), host(w), host(b), 1e-5)
        assert (np.abs(host(y) - want) <= tolerance(host(x), host(w), n, m, r)).all()
        gx, gw, gb = F.layer_norm_backward(g, x, w, mean, rstd)
        G = host(g)
        nn = (host(x) - host(mean)[:, None]) * host(rstd)[:, None]
        # sums of R / 1024 to R / 256 terms in each thread, then 256
        bound = 300 * U * (np.abs(G) * (np.abs(nn) + 1)).sum(0)
        assert (np.abs(host(gw) - (G * nn).sum(0)) <= bound).all()
        assert (np.abs(host(gb) - G.sum(0)) <= 300 * U * np.abs(G).sum(0)).all()


def test_rows_of_one_value_and_not_finite_ones():
    x = torch.randn(6, 200, device="cuda")
    x[1] = 3.25                      # no deviation: the shift, and a finite rstd
    x[3, 7] = float("inf")
    x[4, 9] = float("nan")
    b = torch.randn(200, device="cuda")
    y, mean, rstd = F.layer_norm(x, None, b, extras=True)
    assert torch.equal(y[1], b) and abs(float(rstd[1]) * 1e-5 ** 0.5 - 1) < 1e-6
    assert torch.isnan(y[3]).all() and torch.isnan(y[4]).all()
    clean = F.layer_norm(x[[0, 2, 5]], None, b)
    assert torch.equal(y[[0, 2, 5]], clean)
    # a large common offset: the deviations are taken from the mean
    z = (torch.randn(3, 300, device="cuda") + 4096.0).to(torch.float32)
    want = exact(host(z), 1.0, 0.0, 1e-5)[0]
    # (x is exact; the mean is off by 42 U of 4096 = 0.01 of a deviation of 1)
    assert np.abs(host(F.layer_norm(z)) - want).max() <= 42 * U * 4096 * 1.2 * 2


def test_shapes_and_kinds():
    rng = np.random.default_rng(7)
    x, w, b = data(rng, 24, 100, "f32")
    y, mean, rstd = F.layer_norm(x.view(2, 3, 4, 100), Parameters(w), Parameters(b), extras=True)
    assert y.shape == (2, 3, 4, 100) and mean.shape == rstd.shape == (2, 3, 4)
    flat = F.layer_norm(x, w, b)
    assert torch.equal(y.view(24, 100), flat)
    g = torch.randn(2, 3, 4, 100, device="cuda")
    gx, gw, gb = F.layer_norm_backward(g, x.view(2, 3, 4, 100), w, mean, rstd)
    assert gx.shape == g.shape and gw.shape == gb.shape == (100,)
    h = F.layer_norm(x.cpu().numpy(), w.cpu().numpy(), b.cpu().numpy())
    assert isinstance(h, np.ndarray) and np.array_equal(h, flat.cpu().numpy())
    one = F.layer_norm(x[0], w, b)
    assert one.shape == (100,) and torch.equal(one, flat[0])
    wide = torch.randn(24, 203, device="cuda")
    assert torch.equal(F.layer_norm(wide[:, 3:103], w, b),
                       F.layer_norm(wide[:, 3:103].contiguous(), w, b))
    e, m, r = F.layer_norm(x[:0], w, b, extras=True)
    assert e.shape == (0, 100)
    gx, gw, gb = F.layer_norm_backward(x[:0], x[:0], w, m, r)
    assert gx.shape == (0, 100) and not gw.any() and not gb.any()


def test_one_row_as_an_array():
    """An array of one dimension there and back: the row's own gradients."""
    x, w, b = data(np.random.default_rng(9), 1, 100, "f32")
    g = torch.randn(1, 100, device="cuda")
    h = [t.cpu().numpy() for t in (x[0], w, b, g[0])]
    y, mean, rstd = F.layer_norm(h[0], h[1], h[2], extras=True)
    want = F.layer_norm(x, w, b, extras=True)
    got = F.layer_norm_backward(h[3], h[0], h[1], mean, rstd)
    for a, c in zip((y, *got), (want[0], *F.layer_norm_backward(g, x, w, *want[1:]))):
        assert isinstance(a, np.ndarray) and np.array_equal(a, c.cpu().numpy().reshape(100))


def test_captured_and_on_another_stream():
    x, w, b = data(np.random.default_rng(8), 300, 784, "bf16")
    g = torch.randn(300, 784, device="cuda").bfloat16()

    def both():
        y, mean, rstd = F.layer_norm(x, w, b, extras=True)
        return (y, *F.layer_norm_backward(g, x, w, mean, rstd))

    want = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both()
    side.synchronize()
    assert all(torch.equal(a, e) for a, e in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for k in range(3):
        x.copy_(torch.randn_like(x))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, e) for a, e in zip(out, both()))
