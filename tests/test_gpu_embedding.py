"""Embedding lookup and its gradient against 64-bit sums."""
import numpy as np
import pytest
import torch

from novann_amd import functional as F
from novann_amd.module import Parameters, QuantizedParameters
from tests.token_oracle import HALF_MIN, HALF_ULP, TORCH, floats, host, table

pytestmark = pytest.mark.gpu


def zipf(rng, n, V):
    return np.clip(np.exp(rng.random(n) * np.log(V)).astype(np.int64) - 1, 0, V - 1)


@pytest.mark.parametrize("wdtype", ["f32", "bf16", "f16", "e4m3", "e5m2", "e2m1"])
@pytest.mark.parametrize("out", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("V,D,shape", [(97, 64, (5, 7)), (33, 37, (19,)), (1, 8, (1,)),
                                       (300, 1001, (2, 3, 2)), (11, 1, (4,))])
def test_lookup(wdtype, out, V, D, shape):
    rng = np.random.default_rng(V + D)
    w, _ = table(rng, V, D, wdtype)
    t = rng.integers(0, V, shape)
    y = F.embedding(torch.from_numpy(t).cuda(), w, factor=1.7, out_dtype=out)
    # one fp32 product of the two factors, one with each decoded element, one
    # rounding: the same bits
    if wdtype in ("e4m3", "e5m2", "e2m1"):
        one = QuantizedParameters(w.codes, w.shape, w.dtype, torch.ones_like(w.scale)).dequantize()
        a = (w.scale * np.float32(1.7)).reshape(())
    else:
        one, a = w.data.float(), torch.tensor(1.7, device="cuda")
    want = (one[torch.from_numpy(t).cuda()] * a).to(TORCH[out])
    assert y.shape == (*shape, D) and y.dtype == TORCH[out]
    assert torch.equal(y, want)


def test_lookup_int32_numpy_and_outside_ids():
    rng = np.random.default_rng(0)
    w, d = table(rng, 50, 24, "f32")
    t = rng.integers(0, 50, 9)
    y = F.embedding(t, w)
    assert isinstance(y, np.ndarray) and np.array_equal(y, d[t].astype(np.float32))
    ids = torch.tensor([3, -1, 50, 49], dtype=torch.int32, device="cuda")
    y = F.embedding(ids, w).cpu().numpy()
    assert np.array_equal(y[[0, 3]], d[[3, 49]].astype(np.float32))
    assert np.isnan(y[1:3]).all()
    assert F.embedding(torch.zeros(0, dtype=torch.int64, device="cuda"), w).shape == (0, 24)


def check_gradient(t, g, got, V, factor, old=None):
    """|error| <= (additions + 2) half-ulps of the summed magnitudes (fp32 sums
    in any order, the factor, an old value), and one rounding of the result."""
    name = {v: k for k, v in TORCH.items()}[got.dtype]
    g64 = host(g).reshape(-1, g.shape[-1])
    t = t.reshape(-1)
    ok = (t >= 0) & (t < V)
    want, size = np.zeros((V, g64.shape[1])), np.zeros((V, g64.shape[1]))
    np.add.at(want, t[ok], g64[ok])
    np.add.at(size, t[ok], np.abs(g64[ok]))
    count = np.bincount(t[ok], minlength=V)[:, None]
    want, size = want * factor, size * abs(factor)
    if old is not None:
        want, size = want + old, size + np.abs(old)
    bound = (count + 2) * 2.0 ** -24 * size + HALF_ULP[name] * 1.01 * np.abs(want) + HALF_MIN[name]
    bad = np.abs(host(got) - want) > bound
    assert not bad.any(), (bad.sum(), np.argwhere(bad)[:3])


@pytest.mark.parametrize("gdtype,odtype", [("f32", "f32"), ("bf16", "f32"), ("f16", "f32"),
                                           ("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16")])
@pytest.mark.parametrize("n,V,D", [(1, 1, 1), (1, 700, 96), (15, 3, 33), (17, 2, 520), (257, 70000, 20),
                                   (2048, 513, 24), (2049, 511, 36), (5000, 300, 129)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_gradient(gdtype, odtype, n, V, D, accumulate):
    rng = np.random.default_rng(n + V + D)
    t = zipf(rng, n, V)
    g = floats(rng, (n, D), gdtype)
    old = floats(rng, (V, D), odtype) if accumulate else None
    out = old.clone() if accumulate else torch.full((V, D), float("nan"), device="cuda",
                                                    dtype=TORCH[odtype])
    ids = torch.from_numpy(t).cuda()
    got = F.embedding_backward(g, ids, (V, D), factor=0.5, out=out, accumulate=accumulate)
    assert got is out
    check_gradient(t, g, got, V, 0.5, host(old) if accumulate else None)
    if not accumulate:
        again = F.embedding_backward(g, ids.int(), (V, D), factor=0.5, out=torch.empty_like(out))
        assert torch.equal(got, again)


@pytest.mark.parametrize("kind", ["one token", "ascending", "outside", "two tokens"])
@pytest.mark.parametrize("n", [1, 16, 33, 4097, 20000])
def test_gradient_orders(kind, n):
    V, D = 6000, 72
    rng = np.random.default_rng(n)
    t = {"one token": np.full(n, 4999), "ascending": np.arange(n) % V,
         "outside": rng.choice(np.array([-1, 5, V, V + 7, -(1 << 40), 1 << 40]), n),
         "two tokens": rng.integers(0, 2, n) * (V - 1)}[kind]
    g = floats(rng, (n, D), "bf16")
    got = F.embedding_backward(g, torch.from_numpy(t).cuda(), (V, D))
    check_gradient(t, g, got, V, 1.0)


@pytest.mark.parametrize("n,V,D", [(512, 300, 72), (513, 300, 72), (512, 90, 1032), (300, 700, 130),
                                   (400, 700, 130), (1000, 64, 16), (3000, 5000, 40),
                                   (16, 70000, 512), (600, 70000, 512)])
def test_gradient_of_few_tokens_and_large_tables(n, V, D):
    rng = np.random.default_rng(n + D)
    g = floats(rng, (n, D), "bf16")
    for t in (np.full(n, V - 1), rng.integers(-1, V + 1, n), rng.integers(0, 3, n) * (V // 3),
              np.arange(n)[::-1] % V):
        out = torch.full((V, D), float("nan"), device="cuda")
        F.embedding_backward(g, torch.from_numpy(t.copy()).cuda(), (V, D), out=out)
        check_gradient(t, g, out, V, 1.0)
        twice = F.embedding_backward(g, torch.from_numpy(t.copy()).cuda(), (V, D), out=out.clone(),
                                     accumulate=True)
        assert torch.equal(twice, out + out)


def test_gradient_is_the_difference_of_the_lookup():
    rng = np.random.default_rng(3)
    V, D, n = 40, 12, 100
    w = rng.standard_normal((V, D))
    t = rng.integers(0, V, n)
    g = floats(rng, (n, D), "f32")
    grad = host(F.embedding_backward(g, torch.from_numpy(t).cuda(), (V, D), factor=1.5))
    d = rng.standard_normal((V, D))
    up, down = ((1.5 * (w + s * 1e-3 * d)[t] * host(g)).sum() for s in (1, -1))
    # the lookup is linear: its difference quotient is its derivative
    assert abs((up - down) / 2e-3 - (grad * d).sum()) <= 1e-5 * np.abs(grad * d).sum()


def test_views_and_streams():
    rng = np.random.default_rng(5)
    V, D, n = 301, 40, 777
    big = floats(rng, (n, 2 * D + 1), "bf16")
    g = big[:, 1:D + 1]  # strided, unaligned
    t = torch.from_numpy(rng.integers(0, V, 2 * n)).cuda()[::2]
    w = floats(rng, (2 * V, D), "f16")[1::2]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = F.embedding(t, Parameters(w), out_dtype="f16")
        gw = F.embedding_backward(g, t, Parameters(w))
    s.synchronize()
    assert torch.equal(y, w[t])
    check_gradient(t.cpu().numpy(), g, gw, V, 1.0)


def test_nan_and_inf_stay_in_their_rows():
    t = torch.tensor([4, 2, 4, 7], device="cuda")
    g = torch.ones(4, 16, device="cuda")
    g[0, 3], g[1, 5], g[3, 0] = float("nan"), float("inf"), -float("inf")
    got = F.embedding_backward(g, t, (9, 16)).cpu().numpy()
    assert np.isnan(got[4, 3]) and got[2, 5] == np.inf and got[7, 0] == -np.inf
    assert np.isfinite(np.delete(got, [2, 4, 7], 0)).all() and (~np.isfinite(got)).sum() == 3


def test_graph_replays():
    rng = np.random.default_rng(9)
    V, D, n = 900, 64, 3000
    t = torch.from_numpy(zipf(rng, n, V)).cuda()
    w, _ = table(rng, V, D, "e4m3")
    g = floats(rng, (n, D), "bf16")
    F.embedding_backward(g, t, w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = F.embedding(t, w)
        gw = F.embedding_backward(g, t, w)
    for seed in range(3):
        t.copy_(torch.from_numpy(zipf(np.random.default_rng(seed), n, V)))
        g.copy_(floats(np.random.default_rng(seed), (n, D), "bf16"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, F.embedding(t, w))
        assert torch.equal(gw, F.embedding_backward(g, t, w))
