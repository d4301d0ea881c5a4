"""grad_norm and clip_grad_norm against 64-bit sums.

The squares are summed in fp64, so the fp32 norm is within one ulp (2^-23,
relative) of the true one; the factor takes three more fp32 roundings, the
product one, the store one of the output's type."""
import numpy as np
import pytest
import torch

from novann_amd import optim
from novann_amd.module import Parameters, QuantizedParameters
from tests.token_oracle import HALF_MIN, HALF_ULP, TORCH, floats, host

pytestmark = pytest.mark.gpu


def true_norm(grads):
    return np.sqrt(sum((host(g) ** 2).sum() for g in grads))


def check(grads, outs, norm, max_norm, eps=1e-6):
    n = true_norm(grads)
    assert abs(float(norm) - n) <= 2.0 ** -23 * n
    coef = min(1.0, max_norm / (n + eps))
    for g, o in zip(grads, outs):
        name = {v: k for k, v in TORCH.items()}.get(o.dtype, "f32")
        want = host(g) * coef
        u = 6 * 2.0 ** -24 + HALF_ULP[name] * 1.01
        assert (np.abs(host(o) - want) <= u * np.abs(want) + HALF_MIN[name]).all()


@pytest.mark.parametrize("gdtype,odtype", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"),
                                           ("bf16", "f32"), ("f32", "bf16"), ("f16", "f32")])
@pytest.mark.parametrize("sizes", [(1,), (7,), (4096,), (4097, 3, 0, 8191), (100003, 64, 5),
                                   tuple(range(1, 230)), (1 << 22,)])
@pytest.mark.parametrize("max_norm", [0.5, 1e6])
def test_clip(gdtype, odtype, sizes, max_norm):
    rng = np.random.default_rng(len(sizes))
    grads = [floats(rng, (n,), gdtype, 0.3) for n in sizes]
    outs = [torch.full((n,), float("nan"), device="cuda", dtype=TORCH[odtype]) for n in sizes]
    norm = optim.clip_grad_norm(grads, max_norm, out=outs)
    check(grads, outs, norm, max_norm)
    assert abs(float(optim.grad_norm(grads)) - true_norm(grads)) <= 2.0 ** -23 * true_norm(grads)
    before = [g.clone() for g in grads]
    optim.clip_grad_norm(grads, max_norm)  # in place
    check(before, grads, norm, max_norm)


def test_mixed_types_views_and_float64():
    rng = np.random.default_rng(1)
    flat = floats(rng, (5000,), "f32")
    grads = [flat[1:2000], flat[2001:2004], floats(rng, (33, 65), "bf16")[:, 1:],
             floats(rng, (129,), "f16")[1:], torch.randn(77, 5, device="cuda").double(),
             torch.randn(40, 60, device="cuda").t()]
    before = [g.clone() for g in grads]
    rest = flat[2000].clone(), flat[2004:].clone()
    norm = optim.clip_grad_norm(grads, 2.0)
    check(before, grads, norm, 2.0)
    assert torch.equal(flat[2000], rest[0]) and torch.equal(flat[2004:], rest[1])
    # float64 keeps what a double product gives (the factor itself is fp32)
    n = true_norm(before)
    assert np.allclose(host(grads[4]), host(before[4]) * 2.0 / n, rtol=1e-6, atol=0)


def test_parameters_and_arrays():
    rng = np.random.default_rng(2)
    a = Parameters(np.zeros((6, 5), np.float32))
    a.grad = rng.standard_normal((6, 5)).astype(np.float32)
    b = Parameters(np.zeros(4))  # float64, as BatchNorm's gamma
    b.grad = rng.standard_normal(4)
    c = QuantizedParameters.from_float(rng.standard_normal((8, 16)).astype(np.float32), "e4m3")
    c.grad = floats(rng, (8, 16), "f32")
    d = Parameters(np.zeros(3, np.float32))
    d.grad = None
    before = [torch.from_numpy(a.grad.copy()), torch.from_numpy(b.grad.copy()), c.grad.clone()]
    held = a.grad
    norm = optim.clip_grad_norm([a, b, c, d], 1.0)
    assert a.grad is held
    check(before, [torch.from_numpy(a.grad), torch.from_numpy(b.grad), c.grad], norm, 1.0)


def test_range_of_fp32():
    """The squares of the largest and smallest fp32 gradients keep their size."""
    for v in (1e38, 1e-38, 1e-44):
        g = torch.full((1000,), v, device="cuda")
        n = float(optim.grad_norm([g]))
        want = float(np.float32(v)) * np.sqrt(1000)
        if want < 3e38:
            assert abs(n - want) <= 2.0 ** -23 * want + 2.0 ** -149
        else:
            assert n == np.inf


def test_nan_inf_zero_and_nothing():
    g = [torch.ones(5000, device="cuda"), torch.ones(3, device="cuda")]
    g[1][1] = float("nan")
    norm = optim.clip_grad_norm(g, 1.0)
    assert torch.isnan(norm) and all(torch.isnan(x).all() for x in g)
    g = [torch.ones(10, device="cuda")]
    g[0][2] = float("inf")
    norm = optim.clip_grad_norm(g, 1.0)
    assert float(norm) == np.inf
    assert torch.isnan(g[0][2]) and not g[0][:2].any()
    z = [torch.zeros(100, device="cuda")]
    assert float(optim.clip_grad_norm(z, 1.0)) == 0.0 and not z[0].any()
    assert float(optim.clip_grad_norm([], 1.0)) == 0.0
    assert float(optim.grad_norm([torch.zeros(0, device="cuda")])) == 0.0
    one = [torch.full((4,), 3.0, device="cuda")]
    optim.clip_grad_norm(one, 0.0)
    assert not one[0].any()


def test_stream_and_graph():
    rng = np.random.default_rng(4)
    grads = [floats(rng, (n,), "bf16") for n in (70000, 9, 12345)]
    outs = [torch.empty(g.shape, device="cuda") for g in grads]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        norm = optim.clip_grad_norm(grads, 1.0, out=outs)
    s.synchronize()
    check(grads, outs, norm, 1.0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = optim.clip_grad_norm(grads, 1.0, out=outs)
    for seed in range(3):
        for g in grads:
            g.copy_(floats(np.random.default_rng(seed), g.shape, "bf16"))
        graph.replay()
        torch.cuda.synchronize()
        check(grads, outs, norm, 1.0)
        again = [torch.empty_like(o) for o in outs]
        assert torch.equal(norm, optim.clip_grad_norm(grads, 1.0, out=again))
        assert all(torch.equal(a, b) for a, b in zip(outs, again))


def test_a_shared_parameter_counts_once():
    p = Parameters(np.zeros((2, 3), np.float32))
    p.grad = np.full((2, 3), 2.0, np.float32)
    assert abs(float(optim.grad_norm([p, p])) - np.sqrt(24)) <= 2.0 ** -23 * np.sqrt(24)
    optim.clip_grad_norm([p, p], np.sqrt(24) / 2, eps=0.0)
    assert np.allclose(p.grad, 1.0, rtol=6 * 2.0 ** -24, atol=0)
