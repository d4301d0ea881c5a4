"""linear_cross_entropy_backward with a gradient for each row: no row's gradient
changes what another row gets.

With p = softmax - onehot and u the rounding of the products' 16-bit type, a row of
grad_x is off by (u + 2 e) |g| |p| |W| and its own rounding, as in the tests of equal
rows.  In f16, p of a row at most 2^-20 below the largest is kept to 2^-28 (a
product of f16 range 2^-25 that has 14 - 10 binary places to spare), and x, for
grad_W, to 2^-15 (10 places down): |g| 2^-28 |W| and |g| (2^-28 |x| + 2^-15 |p|) more."""
import numpy as np
import pytest
import torch

from novann_amd import functional as F
from novann_amd.module import Parameters
from tests.token_oracle import (HALF_MIN, HALF_ULP, TORCH, cross_entropy, cross_entropy_grads,
                                floats, host, table)

pytestmark = pytest.mark.gpu


def logit_error(x, w, lse):
    s = (np.abs(x) @ np.abs(w).T).max()
    return np.sqrt(x.shape[1]) * 2.0 ** -23 * s + 2.0 ** -20 * (1 + np.abs(lse).max())


def run(N, D, V, wdtype, xdtype, up, std=1.0, lift=0.0):
    """x, the table in 64 bits, targets, the gradients for the upstream ones."""
    rng = np.random.default_rng(N + D + V)
    if lift:  # a table of values around `lift`
        w = torch.from_numpy((lift + rng.standard_normal((V, D)) / 4).astype(np.float32)).cuda()
        w = w.to(TORCH[wdtype])
        w, w64 = Parameters(w), host(w)
    else:
        w, w64 = table(rng, V, D, wdtype, 1.5 / np.sqrt(D))
    x, t = floats(rng, (N, D), xdtype, std), rng.integers(0, V, N)
    t[1] = -100
    ids = torch.from_numpy(t).cuda()
    _, lse = F.linear_cross_entropy(x, w, ids, reduction="none", extras=True)
    gx, gw = F.linear_cross_entropy_backward(x, w, ids, lse, grad=torch.from_numpy(up).cuda(),
                                             reduction="none", weight_grad_dtype="f32")
    return host(x), w64, t, host(gx), host(gw)


def bounds(x, w, t, up, xdtype):
    """(grad_x, its bound, grad_W, its bound) for finite row gradients."""
    g = np.where(t == -100, 0.0, up.astype(np.float64))
    xs = np.where((t != -100)[:, None], x, 0.0)
    p, _, _ = cross_entropy_grads(xs, w, t, np.ones(len(t)))
    rel = HALF_ULP[xdtype] * 1.01 + 2 * logit_error(xs, w, cross_entropy(xs, w, t)[1])
    small, lost = (2.0 ** -28, 2.0 ** -15) if xdtype == "f16" else (0.0, 0.0)
    a = np.abs(g)[:, None]
    want_x, want_w = (g[:, None] * p) @ w, (g[:, None] * p).T @ xs
    bx = a * (rel * np.abs(p) + small * (g != 0)[:, None]) @ np.abs(w)
    bw = (a * (rel * np.abs(p) + small)).T @ np.abs(xs) + lost * (a * np.abs(p)).sum(0)[:, None]
    return (want_x, bx + HALF_ULP[xdtype] * 1.01 * np.abs(want_x) + HALF_MIN[xdtype], want_w,
            bw + 2.0 ** -23 * np.abs(want_w) + HALF_MIN["f32"])


@pytest.mark.parametrize("xdtype", ["bf16", "f16"])
@pytest.mark.parametrize("N,D,V,wdtype", [(40, 48, 530, "e4m3"), (300, 130, 3000, "bf16"),
                                          (16, 2048, 300, "e5m2")])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_one_row_that_is_not_finite(N, D, V, wdtype, xdtype, bad):
    up = (np.random.default_rng(1).standard_normal(N) / 30).astype(np.float32)
    up[1] = np.nan  # (an ignored row's counts for nothing)
    up[2] = 0.0
    up[5] = bad
    x, w, t, gx, gw = run(N, D, V, wdtype, xdtype, up)
    if wdtype == "bf16" and xdtype == "f16":  # (the table as the products take it)
        w = host(torch.from_numpy(w.astype(np.float32)).to(torch.float16))
    finite = np.where(np.isfinite(up), up, 0.0)
    want_x, bx, _, _ = bounds(x, w, t, finite, xdtype)
    others = np.arange(N) != 5
    assert (np.abs(gx - want_x)[others] <= bx[others]).all()
    assert not gx[1:3].any()
    one = np.zeros(N, np.float32)
    one[5] = 1.0
    row_x, bx, row_w, bw = bounds(x, w, t, one, xdtype)
    if np.isnan(bad):
        assert np.isnan(gx[5]).all() and np.isnan(gw).all()
        return
    # an infinity keeps the sign that the row's own gradient has
    sure = np.abs(row_x[5]) > 2 * bx[5]
    assert (gx[5][sure] == bad * np.sign(row_x[5][sure])).all()
    sure = np.abs(row_w) > 2 * bw
    assert sure.any() and (gw[sure] == bad * np.sign(row_w[sure])).all()
    assert not np.isfinite(gw).any()


@pytest.mark.parametrize("xdtype", ["bf16", "f16"])
@pytest.mark.parametrize("N,D,V", [(41, 24, 50000), (200, 264, 3001), (41, 2048, 200)])
def test_rows_of_very_different_gradients(N, D, V, xdtype):
    """Loss-scaled upstreams from 512 down to 2^-20 of it: every row's gradient is as
    near to its own size as when all are equal.  The table's values have one sign and x
    is small: the softmax's many values, nearly equal, add up."""
    rng = np.random.default_rng(3)
    up = (512 * 2.0 ** (-20 * np.arange(N) / (N - 1)) * rng.choice([-1, 1], N)).astype(np.float32)
    x, w, t, gx, gw = run(N, D, V, xdtype, xdtype, up, std=0.02, lift=1.0)
    want_x, bx, want_w, bw = bounds(x, w, t, up, xdtype)
    bad = np.abs(gx - want_x) > bx
    assert not bad.any(), sorted(set(np.argwhere(bad)[:, 0]))
    bad = np.abs(gw - want_w) > bw
    assert not bad.any(), (bad.sum(), np.argwhere(bad)[:3])


def test_gradients_of_the_whole_range():
    """Upstreams from 2^-100 to 2^100, zeros among them, in bf16."""
    N, D, V = 60, 40, 300
    up = (2.0 ** np.linspace(-100, 100, N)).astype(np.float32)
    up[::7] = 0.0
    x, w, t, gx, gw = run(N, D, V, "e4m3", "bf16", up)
    want_x, bx, want_w, bw = bounds(x, w, t, up, "bf16")
    assert (np.abs(gx - want_x) <= bx).all() and (np.abs(gw - want_w) <= bw).all()
    x, w, t, gx, gw = run(N, D, V, "e4m3", "bf16", np.zeros(N, np.float32))
    assert not gx.any() and not gw.any()


@pytest.mark.parametrize("grad", [np.float32(0.25), np.float64(0.25), 0.25, np.array(0.25),
                                  np.array([0.25], np.float32)])
def test_numbers_as_upstream_gradients(grad):
    """The loss of arrays is an np.float32; so may its gradient be."""
    rng = np.random.default_rng(5)
    x, w = rng.standard_normal((6, 16)).astype(np.float32), rng.standard_normal((9, 16))
    w, t = Parameters(w.astype(np.float32)), rng.integers(0, 9, 6)
    _, lse = F.linear_cross_entropy(x, w, t, extras=True)
    gx, gw = F.linear_cross_entropy_backward(x, w, t, lse, grad=grad)
    full_x, full_w = F.linear_cross_entropy_backward(x, w, t, lse)
    # (a quarter is exact in every step)
    assert np.array_equal(gx, 0.25 * full_x) and np.array_equal(gw, 0.25 * full_w)
    if np.ndim(grad) == 0:
        rows = F.linear_cross_entropy_backward(x, w, t, lse, grad=grad, reduction="none")[0]
        want = F.linear_cross_entropy_backward(x, w, t, lse, reduction="sum")[0]
        assert np.array_equal(rows, 0.25 * want)
