"""linear_cross_entropy and its gradients against the formulas in 64 bits.

Bounds, each derived before it was first run: with S the largest sum of
|x w| in a logit, D products summed in fp32 leave a logit off by at most about
sqrt(D) 2^-23 S (rounding errors of random sign, doubled), and exp, log and the
change of base by 2^-20 (1 + |lse|).  A gradient's softmax is off by twice that,
relatively, and by one rounding to the products' type (u), so an element of
grad_x by at most (u + 2 e) |P| |W| (a matrix product of magnitudes); its own
rounding comes on top.  f16 keeps P with a factor of 2^14: what falls under its
subnormals is at most 2^-39 in size."""
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


def inputs(N, D, V, wdtype, xdtype, seed=0, ignore=0.1):
    rng = np.random.default_rng(seed + N + D + V)
    w, w64 = table(rng, V, D, wdtype, 1.5 / np.sqrt(D))
    t = rng.integers(0, V, N)
    x = floats(rng, (N, D), xdtype) + torch.from_numpy(
        (3 * rng.random((N, 1)) * w64[t]).astype(np.float32)).cuda().to(TORCH[xdtype])
    t[rng.random(N) < ignore] = -100
    return x, w, w64, t


CASES = [(1, 64, 130, "e4m3", "bf16"), (1, 8, 1, "e4m3", "bf16"), (3, 37, 1001, "e2m1", "f16"),
         (65, 128, 257, "e5m2", "f16"), (129, 200, 300, "bf16", "bf16"),
         (200, 96, 9000, "e4m3", "bf16"), (130, 515, 700, "f16", "f16"),
         (40, 64, 20001, "e2m1", "bf16"), (257, 256, 512, "e4m3", "f16"),
         (16, 1024, 2048, "bf16", "bf16"), (300, 1, 50, "e4m3", "bf16"),
         (33, 72, 18000, "bf16", "f16"), (64, 64, 640, "f16", "bf16"),
         (600, 640, 2600, "e4m3", "bf16"), (513, 392, 1030, "e5m2", "f16")]


def rounded(w64, wdtype, ct):
    """The table as the products take it."""
    if wdtype in ("e4m3", "e5m2", "e2m1") or wdtype == ct:
        return w64
    return host(torch.from_numpy(w64.astype(np.float32)).to(TORCH[ct]))


@pytest.mark.parametrize("N,D,V,wdtype,xdtype", CASES)
def test_loss(N, D, V, wdtype, xdtype):
    x, w, w64, t = inputs(N, D, V, wdtype, xdtype)
    ids = torch.from_numpy(t).cuda()
    each, lse = F.linear_cross_entropy(x, w, ids, reduction="none", extras=True)
    x64, w64 = host(x), rounded(w64, wdtype, xdtype)
    want, want_lse, _ = cross_entropy(x64, w64, t)
    e = logit_error(x64, w64, want_lse)
    assert np.abs(host(lse) - want_lse).max() <= e
    assert np.abs(host(each) - want).max() <= 2 * e
    assert (host(each)[t == -100] == 0).all()
    n = max(1, (t != -100).sum())
    mean = F.linear_cross_entropy(x, w, ids)
    assert mean.shape == () and abs(float(mean) - want.sum() / n) <= 2 * e
    total = F.linear_cross_entropy(x, w, ids.int(), reduction="sum")
    assert abs(float(total) - want.sum()) <= 2 * e * n


def check_grads(x, w, w64, t, f, gx, gw, xdtype):
    x64 = np.where((t != -100)[:, None], host(x), 0.0)
    P, want_x, want_w = cross_entropy_grads(x64, w64, t, f)
    _, lse, _ = cross_entropy(x64, w64, t)
    ct = "f16" if xdtype == "f16" else "bf16"
    rel = HALF_ULP[ct] * 1.01 + 2 * logit_error(x64, w64, lse)
    # values of P under the subnormals of f16 (2^-25 with the factor taken off)
    floor = np.abs(f).max() * (2.0 ** -39 if ct == "f16" else 0.0)
    for got, want, size, few in ((gx, want_x, np.abs(P) @ np.abs(w64), np.abs(w64).sum(0)),
                                 (gw, want_w, np.abs(P).T @ np.abs(x64), np.abs(x64).sum(0))):
        name = {v: k for k, v in TORCH.items()}[got.dtype]
        bound = rel * size + HALF_ULP[name] * 1.01 * np.abs(want) + HALF_MIN[name] + floor * few
        bad = np.abs(host(got) - want) > bound
        assert not bad.any(), (bad.sum(), np.argwhere(bad)[:3])


@pytest.mark.parametrize("N,D,V,wdtype,xdtype", CASES)
def test_gradients(N, D, V, wdtype, xdtype):
    x, w, w64, t = inputs(N, D, V, wdtype, xdtype)
    w64 = rounded(w64, wdtype, xdtype)
    ids = torch.from_numpy(t).cuda()
    _, lse = F.linear_cross_entropy(x, w, ids, extras=True)
    gx, gw = F.linear_cross_entropy_backward(x, w, ids, lse)
    assert gx.dtype == x.dtype and gw.dtype == x.dtype
    n = max(1, (t != -100).sum())
    check_grads(x, w, w64, t, np.full(N, 1.0 / n), gx, gw, xdtype)
    again = F.linear_cross_entropy_backward(x, w, ids.int(), lse)
    assert torch.equal(gx, again[0]) and torch.equal(gw, again[1])


@pytest.mark.parametrize("xdtype", ["bf16", "f16"])
@pytest.mark.parametrize("wgrad", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_gradient_types_and_upstream(xdtype, wgrad, reduction):
    N, D, V = 70, 104, 530
    x, w, w64, t = inputs(N, D, V, "e4m3", xdtype, seed=1)
    ids = torch.from_numpy(t).cuda()
    rng = np.random.default_rng(2)
    _, lse = F.linear_cross_entropy(x, w, ids, reduction=reduction, extras=True)
    n = max(1, (t != -100).sum())
    if reduction == "none":
        up = torch.from_numpy((rng.standard_normal(N) / 30).astype(np.float32)).cuda()
        up[3] = 0.0
        f = host(up)
    else:
        up = 0.25 if reduction == "mean" else torch.tensor(0.03, device="cuda")
        f = np.full(N, float(up) / (n if reduction == "mean" else 1))
    gx, gw = F.linear_cross_entropy_backward(x, w, ids, lse, grad=up, reduction=reduction,
                                             weight_grad_dtype=wgrad)
    assert gw.dtype == TORCH[wgrad]
    check_grads(x, w, w64, t, f, gx, gw, xdtype)


def test_gradients_are_the_loss_differences():
    N, D, V = 24, 40, 333
    x, w, w64, t = inputs(N, D, V, "e4m3", "bf16", seed=3)
    ids = torch.from_numpy(t).cuda()
    _, lse = F.linear_cross_entropy(x, w, ids, extras=True)
    gx, gw = F.linear_cross_entropy_backward(x, w, ids, lse, weight_grad_dtype="f32")
    x64, n = host(x), (t != -100).sum()
    rng = np.random.default_rng(4)
    for got, at in ((gx, 0), (gw, 1)):
        d = rng.standard_normal(got.shape)
        h = 1e-5
        side = [cross_entropy(x64 + (s * h * d if at == 0 else 0),
                              w64 + (s * h * d if at == 1 else 0), t)[0].sum() / n
                for s in (1, -1)]
        # u of bf16 twice (P and, for gx, the result) on the magnitudes summed
        assert abs((side[0] - side[1]) / (2 * h) - (host(got) * d).sum()) <= \
            4 * 2.0 ** -9 * np.linalg.norm(host(got)) * np.linalg.norm(d)


def test_fp32_and_numpy_operands_round_to_bf16():
    rng = np.random.default_rng(6)
    N, D, V = 30, 48, 90
    x = rng.standard_normal((N, D)).astype(np.float32)
    w = (rng.standard_normal((V, D)) / 7).astype(np.float32)
    t = rng.integers(0, V, N)
    loss, lse = F.linear_cross_entropy(x, Parameters(w), t, extras=True)
    assert isinstance(loss, np.float32) and isinstance(lse, np.ndarray)
    xb, wb = (host(torch.from_numpy(a).to(torch.bfloat16)) for a in (x, w))
    each, want_lse, _ = cross_entropy(xb, wb, t)
    e = logit_error(xb, wb, want_lse)
    assert abs(loss - each.mean()) <= 2 * e and np.abs(lse - want_lse).max() <= e
    gx, gw = F.linear_cross_entropy_backward(x, Parameters(w), t, lse)
    assert gx.dtype == np.float32 and gw.dtype == np.float32
    check_grads(torch.from_numpy(xb), None, wb, t, np.full(N, 1 / N),
                torch.from_numpy(gx), torch.from_numpy(gw), "f32")


def test_ignored_rows_may_hold_anything():
    N, D, V = 140, 64, 300
    x, w, w64, t = inputs(N, D, V, "e4m3", "bf16", seed=7, ignore=0.3)
    ids = torch.from_numpy(t).cuda()
    clean, lse = F.linear_cross_entropy(x, w, ids, extras=True)
    gx, gw = F.linear_cross_entropy_backward(x, w, ids, lse)
    dirty = x.clone()
    dirty[ids == -100] = float("nan")
    dirty[(ids == -100).nonzero()[0], ::2] = float("inf")
    loss, lse2 = F.linear_cross_entropy(dirty, w, ids, extras=True)
    assert torch.equal(loss, clean)
    gx2, gw2 = F.linear_cross_entropy_backward(dirty, w, ids, lse2)
    assert torch.equal(gx, gx2) and torch.equal(gw, gw2)


def test_nothing_to_learn_from():
    N, D, V = 20, 32, 64
    x, w, _, _ = inputs(N, D, V, "e4m3", "bf16")
    ids = torch.full((N,), -100, device="cuda")
    loss, lse = F.linear_cross_entropy(x, w, ids, extras=True)
    assert float(loss) == 0.0
    gx, gw = F.linear_cross_entropy_backward(x, w, ids, lse)
    assert not gx.any() and not gw.any()
    empty = x[:0]
    none = ids[:0]
    loss, lse = F.linear_cross_entropy(empty, w, none, extras=True)
    assert float(loss) == 0.0 and lse.shape == (0,)
    gx, gw = F.linear_cross_entropy_backward(empty, w, none, lse)
    assert gx.shape == (0, D) and gw.shape == (V, D) and not gw.any()
    assert F.linear_cross_entropy(empty, w, none, reduction="none").shape == (0,)


def test_bad_targets_and_values_show():
    N, D, V = 10, 64, 100
    x, w, _, t = inputs(N, D, V, "e4m3", "bf16", ignore=0)
    ids = torch.from_numpy(t).cuda()
    ids[2], ids[5] = V, -7
    each, lse = F.linear_cross_entropy(x, w, ids, reduction="none", extras=True)
    bad = torch.isnan(each).cpu().numpy()
    assert bad.nonzero()[0].tolist() == [2, 5]
    assert torch.isnan(F.linear_cross_entropy(x, w, ids))
    gx, _ = F.linear_cross_entropy_backward(x, w, ids, lse)
    nan = torch.isnan(gx).all(1).cpu().numpy()
    assert nan[[2, 5]].all() and not torch.isnan(gx[[0, 1, 3, 4]]).any()
    x[7, 3] = float("nan")
    ids = torch.from_numpy(t).cuda()
    each = F.linear_cross_entropy(x, w, ids, reduction="none")
    assert torch.isnan(each).cpu().numpy().nonzero()[0].tolist() == [7]


def test_large_and_equal_logits():
    """Logits of thousands (the maximum is taken off before the exponential) and
    rows of equal logits."""
    D, V = 64, 700
    w = torch.zeros(V, D, device="cuda", dtype=torch.bfloat16)
    w[5, 0], w[300, 0], w[699, 0] = 256.0, 256.0, -256.0
    x = torch.zeros(3, D, device="cuda", dtype=torch.bfloat16)
    x[0, 0], x[1, 0] = 32.0, -32.0
    ids = torch.tensor([5, 699, 0], device="cuda")
    each, lse = F.linear_cross_entropy(x, w, ids, reduction="none", extras=True)
    want, want_lse, _ = cross_entropy(host(x), host(w), ids.cpu().numpy())
    assert np.allclose(host(each), want, rtol=0, atol=2.0 ** -20 * 8193)
    assert np.allclose(host(lse), want_lse, rtol=2.0 ** -22)
    gx, gw = F.linear_cross_entropy_backward(x, w, ids, lse, reduction="sum")
    _, wx, ww = cross_entropy_grads(host(x), host(w), ids.cpu().numpy(), np.ones(3))
    assert np.abs(host(gx) - wx).max() <= 2.0 ** -8 * 256 * 2 + 2.0 ** -6
    assert np.abs(host(gw) - ww).max() <= 2.0 ** -8 * 32


def test_views_streams_and_graph():
    N, D, V = 90, 96, 400
    x, w, w64, t = inputs(2 * N, D, V, "e2m1", "f16", seed=8)
    wide = torch.zeros(2 * N, D + 3, device="cuda", dtype=torch.float16)
    wide[:, 1:D + 1] = x
    xs, ids = wide[::2, 1:D + 1], torch.from_numpy(t).cuda()[::2]
    want, lse = F.linear_cross_entropy(xs.contiguous(), w, ids.contiguous(), extras=True)
    gx, gw = F.linear_cross_entropy_backward(xs.contiguous(), w, ids.contiguous(), lse)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got, lse2 = F.linear_cross_entropy(xs, w, ids, extras=True)
        gx2, gw2 = F.linear_cross_entropy_backward(xs, w, ids, lse2)
    s.synchronize()
    assert torch.equal(got, want) and torch.equal(gx, gx2) and torch.equal(gw, gw2)
    fixed, at = xs.contiguous(), ids.contiguous()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, lse2 = F.linear_cross_entropy(fixed, w, at, extras=True)
        gx2, gw2 = F.linear_cross_entropy_backward(fixed, w, at, lse2)
    for seed in range(3):
        fixed.copy_(floats(np.random.default_rng(seed), (N, D), "f16"))
        graph.replay()
        torch.cuda.synchronize()
        want, lse = F.linear_cross_entropy(fixed, w, at, extras=True)
        gx, gw = F.linear_cross_entropy_backward(fixed, w, at, lse)
        assert torch.equal(got, want) and torch.equal(gx, gx2) and torch.equal(gw, gw2)


def test_more_classes_than_one_piece_of_few_rows():
    """A vocabulary of millions: P's row pitch, the pieces and the tiles' counts
    stay within their types."""
    N, D, V = 2, 8, 3_000_001
    rng = np.random.default_rng(11)
    w = floats(rng, (V, D), "bf16", 0.5)
    x = floats(rng, (N, D), "bf16")
    t = np.array([V - 1, 17])
    ids = torch.from_numpy(t).cuda()
    each, lse = F.linear_cross_entropy(x, w, ids, reduction="none", extras=True)
    x64, w64 = host(x), host(w)
    want, want_lse, _ = cross_entropy(x64, w64, t)
    e = logit_error(x64, w64, want_lse)
    assert np.abs(host(each) - want).max() <= 2 * e and np.abs(host(lse) - want_lse).max() <= e
    gx, gw = F.linear_cross_entropy_backward(x, w, ids, lse, reduction="sum",
                                             weight_grad_dtype="f32")
    check_grads(x, w, w64, t, np.ones(N), gx, gw, "bf16")


@pytest.mark.parametrize("N,D,V,wdtype,xdtype", [(5000, 700, 33000, "e4m3", "bf16"),
                                                 (2048, 512, 20011, "e2m1", "f16"),
                                                 (4096, 256, 40000, "bf16", "bf16")])
def test_large_products(N, D, V, wdtype, xdtype):
    """256 x 256 tiles, several pieces with a smaller last one, split sums: the
    bounds of this file with the formulas in float64 on the device."""
    x, w, w64, t = inputs(N, D, V, wdtype, xdtype, seed=5)
    ids = torch.from_numpy(t).cuda()
    loss, lse = F.linear_cross_entropy(x, w, ids, extras=True)
    gx, gw = F.linear_cross_entropy_backward(x, w, ids, lse)
    kept = ids != -100
    n = int(kept.sum())
    X, W = x.double() * kept.unsqueeze(1), torch.from_numpy(w64).cuda()
    l = X @ W.t().contiguous()
    want_lse = torch.logsumexp(l, 1)
    e = float(np.sqrt(D) * 2.0 ** -23 * (X.abs() @ W.abs().t().contiguous()).max()
              + 2.0 ** -20 * (1 + want_lse.abs().max()))
    assert (lse.double() - want_lse).abs()[kept].max() <= e
    at = torch.where(kept, ids, 0).unsqueeze(1)
    each = torch.where(kept, want_lse - l.gather(1, at).squeeze(1), 0.0)
    assert abs(float(loss) - float(each.sum()) / n) <= 2 * e
    P = (l - want_lse.unsqueeze(1)).exp_()
    del l
    P.scatter_add_(1, at, torch.full_like(at, -1, dtype=torch.float64))
    P *= kept.unsqueeze(1) / n
    rel = HALF_ULP[xdtype] * 1.01 + 2 * e
    floor = 2.0 ** -39 / n if xdtype == "f16" else 0.0
    for got, want, size, few in ((gx, P @ W, P.abs() @ W.abs(), W.abs().sum(0)),
                                 (gw, P.t().contiguous() @ X, P.abs().t().contiguous() @ X.abs(),
                                  X.abs().sum(0))):
        bound = rel * size + HALF_ULP[xdtype] * 1.01 * want.abs() + HALF_MIN[xdtype] + floor * few
        bad = (got.double() - want).abs() > bound
        assert not bad.any(), (int(bad.sum()), bad.nonzero()[:3])


@pytest.mark.parametrize("N,D,V,wdtype,xdtype", [(8192, 96, 300, "bf16", "bf16"),
                                                 (20000, 200, 70, "e5m2", "f16"),
                                                 (4100, 1030, 900, "e4m3", "bf16")])
def test_many_tokens_of_few_classes(N, D, V, wdtype, xdtype):
    """grad_W's products are split over the tokens; its types are roundings of one sum."""
    test_large_products(N, D, V, wdtype, xdtype)
    x, w, _, t = inputs(N, D, V, wdtype, xdtype, seed=6)
    ids = torch.from_numpy(t).cuda()
    _, lse = F.linear_cross_entropy(x, w, ids, extras=True)
    full = F.linear_cross_entropy_backward(x, w, ids, lse, weight_grad_dtype="f32")[1]
    for name in ("bf16", "f16"):
        got = F.linear_cross_entropy_backward(x, w, ids, lse, weight_grad_dtype=name)[1]
        assert torch.equal(got, full.to(got.dtype))


@pytest.mark.parametrize("N,D,V,wdtype,xdtype", [(1, 4096, 1280, "e4m3", "bf16"),
                                                 (103, 2560, 1001, "e2m1", "f16"),
                                                 (300, 4090, 258, "bf16", "bf16"),
                                                 (130, 1100, 7, "bf16", "f16")])
def test_wide_rows_of_few_classes(N, D, V, wdtype, xdtype):
    """The logits' products are split over the width."""
    test_loss(N, D, V, wdtype, xdtype)
    test_gradients(N, D, V, wdtype, xdtype)


def test_wide_rows_show_bad_targets_and_ignore_others():
    N, D, V = 40, 2048, 600
    x, w, _, t = inputs(N, D, V, "e4m3", "bf16", seed=9)
    t[0], t[1] = V, -100
    ids = torch.from_numpy(t).cuda()
    each, lse = F.linear_cross_entropy(x, w, ids, reduction="none", extras=True)
    assert torch.isnan(each[0]) and each[1] == 0 and torch.isfinite(each[1:]).all()
    gx, gw = F.linear_cross_entropy_backward(x, w, ids, lse, reduction="none",
                                             grad=torch.ones(N, device="cuda"))
    assert torch.isnan(gx[0]).all() and (gx[1] == 0).all() and torch.isfinite(gx[1:].float()).all()
    assert torch.isnan(gw).all()


@pytest.mark.parametrize("N,D", [(17, 2048), (5, 40)])
def test_one_class(N, D):
    """The softmax is 1 and its gradients 0: what is left of 1 - 1 is the rounding of
    the logit and of lse, twice logit_error of the softmax, times f and the operand."""
    x, w, w64, t = inputs(N, D, 1, "e5m2", "bf16")
    test_loss(N, D, 1, "e5m2", "bf16")
    ids = torch.from_numpy(t).cuda()
    _, lse = F.linear_cross_entropy(x, w, ids, extras=True)
    gx, gw = F.linear_cross_entropy_backward(x, w, ids, lse)
    x64 = np.where((t != -100)[:, None], host(x), 0.0)
    e = 2 * logit_error(x64, w64, cross_entropy(x64, w64, t)[1]) / max(1, (t != -100).sum())
    assert (np.abs(host(gx)) <= 1.01 * e * np.abs(w64)).all()
    assert (np.abs(host(gw)) <= 1.01 * e * np.abs(x64).sum(0)).all()
    assert (host(gx)[t == -100] == 0).all()


def test_few_rows_of_several_pieces():
    """Each piece's logits are split over the width, the last, smaller one further."""
    test_large_products(90, 4096, 18000, "e4m3", "bf16")
