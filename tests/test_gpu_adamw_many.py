"""The AdamW step of many tensors: fp32 states bit for bit as the reference's float32
statements (oracle/optim_ref.py), states in 8 bits bit for bit as tests/adamw_oracle.py
rounds them (the weights beside those to a few units in the last place), and the codes that quantized weights keep."""
import numpy as np
import pytest
import torch

from novann_amd import optim, quant
from novann_amd.module import BlockQuantizedParameters, Parameters, QuantizedParameters
from oracle import optim_ref as OR
from tests import adamw_oracle as A
from tests.token_oracle import TORCH

pytestmark = pytest.mark.gpu
HP = dict(lr=1e-3, betas=(0.9, 0.999), weight_decay=0.02, epsilon=1e-8)
# around a lane's 4 elements, a block of 128, a workgroup's span of 2048, a run
SIZES = [1, 3, 4, 127, 128, 129, 1000, 2047, 2048, 2049, 5000, 16384, 70001]


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def start(rng, n, gdt="f32"):
    """(w, g as stored, m, v) of one tensor."""
    w = rng.standard_normal(n).astype(np.float32)
    g = torch.from_numpy((rng.standard_normal(n) * 0.1).astype(np.float32)).to(TORCH[gdt])
    m = (rng.standard_normal(n) * 0.03).astype(np.float32)
    v = ((rng.random(n) * 0.1) ** 2).astype(np.float32)
    return w, g, m, v


def reference(w, g, m, v, t, decay=True):
    return OR.adamw_step(w, g.float().numpy(), m, v, t, HP["lr"], 0.9, 0.999, 1e-8,
                         HP["weight_decay"], decay)


def same(t, a):
    return np.array_equal(t.cpu().numpy().view(np.uint32), a.view(np.uint32))


@pytest.mark.parametrize("gdt", ["f32", "f16", "bf16"])
def test_fp32_states(gdt):
    rng = np.random.default_rng(1)
    host = [start(rng, n, gdt) for n in SIZES]
    flags = [i % 3 != 0 for i in range(len(host))]
    w, m, v = ([dev(h[k]) for h in host] for k in (0, 2, 3))
    for t in (1, 2, 7):
        optim.adamw_step(w, [h[1].cuda() for h in host], list(zip(m, v)), step=t, decay=flags, **HP)
        host = [(*[a for a in reference(*h, t, f)][:1], h[1], *reference(*h, t, f)[1:])
                for h, f in zip(host, flags)]
        for i, h in enumerate(host):
            assert same(w[i], h[0]) and same(m[i], h[2]) and same(v[i], h[3]), (t, SIZES[i])


def test_more_tensors_than_a_launch_takes():
    rng = np.random.default_rng(2)
    host = [start(rng, int(n)) for n in rng.integers(1, 3000, 131)]
    w, m, v = ([dev(h[k]) for h in host] for k in (0, 2, 3))
    grads = [h[1].cuda() for h in host]
    grads[5] = grads[130] = None
    optim.adamw_step(w, grads, list(zip(m, v)), step=3, **HP)
    for i, h in enumerate(host):
        want = (h[0], h[2], h[3]) if grads[i] is None else reference(*h, 3)
        assert same(w[i], want[0]) and same(m[i], want[1]) and same(v[i], want[2])


def packed(rng, n, first, seed):
    """A State8 on the device and its codes."""
    m = (rng.standard_normal(n) * 0.03 * 10.0 ** rng.uniform(-4, 0, n)).astype(np.float32)
    v = ((rng.random(n) * 0.1 * 10.0 ** rng.uniform(-4, 0, n)) ** 2).astype(np.float32)
    v[rng.random(n) < 0.05] = 0.0
    m[rng.random(n) < 0.05] = 0.0
    codes = A.encode(m, v, first, seed)
    t = [dev(c) for c in codes]
    return optim.State8(t[0].view(torch.float8_e4m3fn), t[1], t[2], t[3]), codes


def near(t, want, before):
    """The step beside 8-bit states: a root and a reciprocal of 1 unit (2^-23) each, three
    constants and five operations rounded once (2^-24): 2^-20.4 of the change, the reference's
    own roundings as much again; w's are 2 here and there."""
    got, want, before = t.double().cpu().numpy(), want.astype(np.float64), before.astype(np.float64)
    return (np.abs(got - want) <= 2.0 ** -19 * np.abs(want - before)
            + 4 * 2.0 ** -24 * (np.abs(want) + np.abs(before))).all()


@pytest.mark.parametrize("gdt", ["f32", "f16", "bf16"])
def test_states_in_8_bits(gdt):
    rng = np.random.default_rng(3)
    host = [start(rng, n, gdt) for n in SIZES]
    firsts = np.concatenate([[0], np.cumsum([128 * A.blocks(n) for n in SIZES])])
    states, codes = zip(*[packed(rng, n, 0, 99) for n in SIZES])
    w = [dev(h[0]) for h in host]
    seed = 12345
    for t in (1, 2):
        optim.adamw_step(w, [h[1].cuda() for h in host], states, step=t, seed=seed + t, **HP)
        new = []
        for i, h in enumerate(host):
            m, v = (a.astype(np.float32) for a in A.decode(*codes[i]))
            got = reference(h[0], h[1], m, v, t)
            want = A.encode(got[1], got[2], int(firsts[i]), seed + t)
            assert near(w[i], got[0], h[0]), SIZES[i]
            s = states[i]
            for a, b in zip((s.m.view(torch.uint8), s.m_exponents, s.v, s.v_exponents), want):
                assert np.array_equal(a.cpu().numpy(), b), SIZES[i]
            new.append(want)
            host[i] = (w[i].cpu().numpy(), *h[1:])
        codes = new


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_decode(dtype):
    rng = np.random.default_rng(4)
    for n in (1, 130, 5003):
        s, codes = packed(rng, n, 0, 7)
        m, v = s.decode(dtype)
        for got, want in zip((m, v), A.decode(*codes)):
            want = torch.from_numpy(want.astype(np.float32)).to(TORCH[dtype])
            assert torch.equal(got.cpu(), want)
    z = optim.State8.zeros(1000)
    assert not any(t.any() for t in z.decode(dtype))


def test_rounding_has_the_right_mean():
    """Over many seeds the mean of the stored states is the fp32 one: its deviation has a
    variance of at most a quarter of a code's gap squared a seed, and 6 of its standard
    deviations are allowed over all elements."""
    rng = np.random.default_rng(5)
    n, seeds = 512, 400
    w, g, _, _ = start(rng, n)
    zero = np.zeros(n, np.float32)
    _, m, v = reference(w, g, zero, zero, 1)
    sums = np.zeros((2, n))
    for s in range(seeds):
        state = optim.State8.zeros(n)
        optim.adamw_step([dev(w)], [g.cuda()], [state], step=1, seed=s, **HP)
        sums += np.stack([t.double().cpu().numpy() for t in state.decode()])
    me, ve = A.encode(m, v, 0, 0)[1::2]
    for got, want, values, e in ((sums[0], np.abs(m), A.E4M3, me), (sums[1], v, A.V, ve)):
        scale = 2.0 ** (A.per_element(e, n) - 127)
        lo = np.searchsorted(values, want / scale, side="right") - 1
        gap = (values[np.minimum(lo + 1, len(values) - 1)] - values[lo]) * scale
        # (a random number has 16 bits: a step of 2^-16 of the gap)
        assert (np.abs(np.abs(got) / seeds - want) <=
                6 * gap / 2 / np.sqrt(seeds) + gap * 2.0 ** -16).all()


def test_a_state_that_decays_does_not_stand_still():
    """v after 500 steps without a gradient: its mean falls as 0.999^t, where nearest codes
    would keep it."""
    n = 4096
    state = optim.State8.zeros(n)
    w = torch.zeros(n, device="cuda")
    hp = dict(HP, lr=0.0)
    g = torch.rand(n, device="cuda") + 0.5
    optim.adamw_step([w], [g], [state], step=1, **hp)
    first = float(state.decode()[1].double().mean())
    zero = torch.zeros_like(g)
    for t in range(2, 502):
        optim.adamw_step([w], [zero], [state], step=t, **hp)
    last = float(state.decode()[1].double().mean())
    # each element's walk has a relative variance below 500 (1/8)^2 / 6 = 1.3; the mean of
    # 4096 is within 6 * 1.14 / 64 = 0.11 of the product
    assert abs(last / first / 0.999 ** 500 - 1) < 0.11


def test_not_finite():
    """A block with an infinity or a NaN decodes to NaN from then on, the others go on."""
    n = 512
    g = torch.full((n,), 0.5, device="cuda")
    g[5], g[300] = float("inf"), float("nan")
    s = optim.State8.zeros(n)
    w = torch.ones(n, device="cuda")
    optim.adamw_step([w], [g], [s], step=1, **HP)
    assert s.m_exponents.tolist()[0] == s.v_exponents.tolist()[0] == 255
    m, v = s.decode()
    bad = torch.zeros(n, dtype=torch.bool, device="cuda")
    bad[:128] = bad[256:384] = True
    assert torch.equal(torch.isnan(m), bad) and torch.equal(torch.isnan(v), bad)
    assert torch.isfinite(w[~bad]).all() and torch.isnan(w[300]) and torch.isfinite(w[6])


def test_small_states():
    """Gradients at the ends of fp32: v's square overflows to a block of NaN, or underflows to
    zero, and m keeps its sign and size."""
    for size in (1e-30, 1e-22, 1e-15, 1e18):
        g = torch.full((256,), size, device="cuda")
        g[::2] *= -1
        s = optim.State8.zeros(256)
        w = torch.zeros(256, device="cuda")
        optim.adamw_step([w], [g], [s], step=1, **HP)
        m, v = (t.cpu().numpy() for t in s.decode())
        _, rm, rv = reference(np.zeros(256, np.float32), g.cpu(), np.zeros(256, np.float32),
                              np.zeros(256, np.float32), 1)
        assert (np.abs(m / rm - 1) <= 1 / 8).all()
        small = rv < 2.0 ** -118
        assert (np.abs(v[~small] / rv[~small] - 1) <= 1 / 8).all()
        assert (v[small] <= 2.0 ** -117.8).all() and ((v[small] > 0) == (rv[small] > 0)).all()


def test_views_keep_their_neighbours():
    """Tensors that start anywhere in a buffer: nothing beside them is written."""
    rng = np.random.default_rng(6)
    for n, off in ((5, 1), (130, 3), (4099, 2)):
        for bits in (32, 8):
            w, g, m, v = start(rng, n, "bf16")
            buf = torch.full((n + 8,), 7.5, device="cuda")
            gbuf = torch.zeros(n + 8, device="cuda", dtype=torch.bfloat16)
            view, gv = buf[off:off + n], gbuf[off:off + n]
            view.copy_(dev(w))
            gv.copy_(g.cuda())
            if bits == 32:
                sb = torch.full((2, n + 8), 3.0, device="cuda")
                state = (sb[0, off:off + n], sb[1, off:off + n])
                state[0].copy_(dev(m)), state[1].copy_(dev(v))
                want = reference(w, g, m, v, 4)
            else:
                sb = torch.full((2, n + 8), 9, dtype=torch.uint8, device="cuda")
                s, codes = packed(rng, n, 0, 5)
                state = optim.State8(sb[0, off:off + n].view(torch.float8_e4m3fn), s.m_exponents,
                                     sb[1, off:off + n], s.v_exponents)
                state.m.view(torch.uint8).copy_(s.m.view(torch.uint8))
                state.v.copy_(s.v)
                m, v = (a.astype(np.float32) for a in A.decode(*codes))
                want = reference(w, g, m, v, 4)
            optim.adamw_step([view], [gv], [state], step=4, **HP)
            assert same(view, want[0]) if bits == 32 else near(view, want[0], w)
            rest = torch.ones(n + 8, dtype=torch.bool)
            rest[off:off + n] = False
            assert (buf.cpu()[rest] == 7.5).all()
            assert (sb.cpu()[:, rest] == (3.0 if bits == 32 else 9)).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_quantized_weights(bits):
    """Per-tensor and block codes beside the step are those of the stepped masters."""
    rng = np.random.default_rng(7)
    shapes = [(130, 257), (128, 128), (300, 40), (64, 1000)]
    for qt in ("e4m3", "e5m2", "e2m1", "b4", "b5"):
        ws = []
        for s in shapes:
            w = (rng.standard_normal(s) * 0.05).astype(np.float32)
            if qt[0] == "b":
                ws.append(BlockQuantizedParameters.from_float(
                    w, "e4m3" if qt == "b4" else "e5m2", keep_master=True,
                    transposed=s != (300, 40)))
            else:
                ws.append(QuantizedParameters.from_float(w, qt, keep_master=True))
        plain = [w.master.clone() for w in ws]
        grads = [torch.randn(p.shape, device="cuda") for p in plain]

        def states():
            return [optim.State8.zeros(p.numel()) if bits == 8 else
                    (torch.zeros_like(p), torch.zeros_like(p)) for p in plain]

        optim.adamw_step(ws, grads, states(), step=1, **HP)
        optim.adamw_step(plain, grads, states(), step=1, **HP)
        for w, p in zip(ws, plain):
            assert torch.equal(w.master, p)
            if qt[0] == "b":
                q, t, _ = quant.make_blocks(p, w.dtype, 128, transposed=True)
                assert torch.equal(w.codes.view(torch.uint8), q.data.view(torch.uint8))
                assert torch.equal(w.exponents, q.exponents)
                if w.codes_t is not None:
                    assert torch.equal(w.codes_t.view(torch.uint8), t.data.view(torch.uint8))
                    assert torch.equal(w.exponents_t, t.exponents)
            else:
                q = quant.quantize(p, qt)
                assert torch.equal(w.codes.view(torch.uint8), q.data.view(torch.uint8))
                assert torch.equal(w.scale, q.scale) and torch.equal(w.amax, q.amax)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("gdt", ["f32", "f16", "bf16"])
def test_weights_that_step_in_tiles(gdt, bits):
    """Many weights with blocks are stepped a tile at a time: the bits of weights without, of
    every state and code, also around values that are not finite."""
    rng = np.random.default_rng(11)
    shapes = [(1000, 1152), (1, 128), (4100, 640), (129, 384), (257, 1024), (130, 100), (300, 200),
              (128, 8)] * 2 + [(8, 128)] * 40
    assert sum(-(-r // 128) * -(-c // 128) for r, c in shapes if c % 128 == 0) >= 256
    ws = [BlockQuantizedParameters.from_float(
        (rng.standard_normal(s) * 0.05).astype(np.float32), "e5m2" if i % 3 == 1 else "e4m3",
        keep_master=True, transposed=i % 4 != 2) for i, s in enumerate(shapes)]
    plain = [w.master.clone() for w in ws]
    grads = [(torch.randn(p.shape, device="cuda") * 1e-2).to(TORCH[gdt]) for p in plain]
    grads[0][500, 300], grads[0][999, 1151], grads[4][256, 0] = float("nan"), float("inf"), -3e38
    flags = [i % 5 != 2 for i in range(len(ws))]
    made = [packed(rng, p.numel(), 0, 3)[0] if bits == 8 else
            (torch.randn_like(p) * 1e-2, torch.rand_like(p) * 1e-4) for p in plain]

    def copies():
        return [optim.State8(*(t.clone() for t in s)) if bits == 8 else
                tuple(t.clone() for t in s) for s in made]

    a, b = copies(), copies()
    for t in (1, 2):
        optim.adamw_step(ws, grads, a, step=t, decay=flags, **HP)
        optim.adamw_step(plain, grads, b, step=t, decay=flags, **HP)
        for i, (w, p) in enumerate(zip(ws, plain)):
            assert torch.equal(w.master.view(torch.int32), p.view(torch.int32)), (t, i)
            for x, y in zip(a[i], b[i]):
                assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)), (t, i)
            q, qt, _ = quant.make_blocks(p, w.dtype, 128, transposed=True)
            assert torch.equal(w.codes.view(torch.uint8), q.data.view(torch.uint8)), (t, i)
            assert torch.equal(w.exponents, q.exponents), (t, i)
            if w.codes_t is not None:
                assert torch.equal(w.codes_t.view(torch.uint8), qt.data.view(torch.uint8)), (t, i)
                assert torch.equal(w.exponents_t, qt.exponents), (t, i)


@pytest.mark.parametrize("qt", ["e4m3", "e5m2", "e2m1"])
def test_a_large_per_tensor_weight(qt):
    """One that is most of a call has a kernel of its own: the bits of a plain weight's step, the
    codes and scale of the stepped master, beside small ones and where it decays or not."""
    big, n = (2048, 2049 if qt != "e2m1" else 2050), 1000
    for flags in ([True, False], [False, True]):
        w = QuantizedParameters.from_float(torch.randn(big, device="cuda") * 0.05, qt,
                                           keep_master=True)
        small = torch.randn(n, device="cuda")
        plain = [w.master.clone(), small.clone()]
        grads = [torch.randn(big, device="cuda"), torch.randn(n, device="cuda")]
        made = [torch.rand_like(t) * 1e-2 for t in (*grads, *grads)]
        a, b = ([(t[0], t[2]), (t[1], t[3])] for t in ([x.clone() for x in made] for _ in range(2)))
        for t in (1, 2):
            optim.adamw_step([w, small], grads, a, step=t, decay=flags, **HP)
            optim.adamw_step(plain, grads, b, step=t, decay=flags, **HP)
            assert torch.equal(w.master, plain[0]) and torch.equal(small, plain[1])
            assert all(torch.equal(x, y) for s, r in zip(a, b) for x, y in zip(s, r))
            q = quant.quantize(w.master, qt)
            assert torch.equal(w.codes.view(torch.uint8), q.data.view(torch.uint8))
            assert torch.equal(w.scale, q.scale) and torch.equal(w.amax, q.amax)


def test_the_class():
    """AdamW over parameters of every kind against the same steps one tensor at a time."""
    rng = np.random.default_rng(8)

    def params():
        r = np.random.default_rng(9)
        a = Parameters(r.standard_normal((5, 7)).astype(np.float32))
        b = Parameters(torch.from_numpy(r.standard_normal(200).astype(np.float32)).cuda())
        b.name = "gamma"
        c = QuantizedParameters.from_float(r.standard_normal((30, 41)).astype(np.float32), "e2m1",
                                           keep_master=True)
        d = BlockQuantizedParameters.from_float(r.standard_normal((130, 60)).astype(np.float32),
                                                keep_master=True)
        e = Parameters(r.standard_normal((1, 9)))
        return [a, b, c, d, e]

    one, many = params(), params()
    opts = [optim.AdamW([p], lr=0.01, weight_decay=0.1) for p in one]
    opt = optim.AdamW(many, lr=0.01, weight_decay=0.1)
    scale = many[2].scale
    for t in range(3):
        for p, q in zip(one, many):
            g = rng.standard_normal(p.shape).astype(np.float32)
            p.grad, q.grad = g, torch.from_numpy(g).cuda()
        many[0].grad = one[0].grad
        many[4].grad = one[4].grad
        for o in opts:
            o.step()
        opt.step()
        if t == 0:
            scale = many[2].scale  # (kept from the first step on: graphs may read it)
        for p, q in zip(one, many):
            x, y = (getattr(r, "master", None) if hasattr(r, "master") else r.data for r in (p, q))
            if isinstance(x, np.ndarray):
                assert np.array_equal(x, y)
            else:
                assert torch.equal(x, y)
        assert torch.equal(one[2].codes, many[2].codes) and torch.equal(one[2].scale, many[2].scale)
        assert many[2].scale.data_ptr() == scale.data_ptr()
        assert torch.equal(one[3].codes.view(torch.uint8), many[3].codes.view(torch.uint8))


def test_shared_parameters_step_once_for_each_name():
    """One tensor named twice steps twice, as one parameter after the other would."""
    w = torch.ones(100, device="cuda")
    p, q = Parameters(w), Parameters(w)
    g = torch.randn(100, device="cuda")
    p.grad = q.grad = g
    optim.AdamW([p, q], lr=0.1).step()
    x = torch.ones(100, device="cuda")
    for _ in range(2):
        s = (torch.zeros(100, device="cuda"), torch.zeros(100, device="cuda"))
        optim.adamw_step([x], [g], [s], lr=0.1, step=1)
    assert torch.equal(w, x)
    # parameters that overlap otherwise, as well
    buf = torch.ones(150, device="cuda")
    a, b = Parameters(buf[:100]), Parameters(buf[50:])
    a.grad = b.grad = g
    optim.AdamW([a, b], lr=0.1).step()
    y = torch.ones(150, device="cuda")
    for part in (y[:100], y[50:]):
        s = (torch.zeros(100, device="cuda"), torch.zeros(100, device="cuda"))
        optim.adamw_step([part], [g], [s], lr=0.1, step=1)
    assert torch.equal(buf, y)


def test_arrays_that_overlap_step_one_after_another():
    """Views of one host array, the second from what the first has left."""
    rng = np.random.default_rng(13)
    base = rng.standard_normal(150).astype(np.float32)
    want = base.copy()
    ps = [Parameters(base[:100]), Parameters(base[50:]), Parameters(base[1:])]
    opt = optim.AdamW(ps, lr=0.1, weight_decay=0.02)
    states = [(np.zeros(p.shape, np.float32),) * 2 for p in ps]
    for t in (1, 2):
        for k, (p, part) in enumerate(zip(ps, (want[:100], want[50:], want[1:]))):
            p.grad = rng.standard_normal(p.shape).astype(np.float32)
            part[...], *states[k] = OR.adamw_step(part.copy(), p.grad, *states[k], t, 0.1, wd=0.02)
        opt.step()
        assert np.array_equal(base, want)


def test_a_refused_step_of_the_class_changes_nothing():
    """One weight's codes on the host: the others are not stepped, and the step is not counted;
    once they are back the step is the first."""
    rng = np.random.default_rng(14)
    bad = BlockQuantizedParameters.from_float(np.ones((8, 16), np.float32), keep_master=True)
    ps = [Parameters(dev(rng.standard_normal(50).astype(np.float32))), bad,
          Parameters(rng.standard_normal(30).astype(np.float32)),
          Parameters(rng.standard_normal(9)), Parameters(rng.standard_normal(9))]
    for p in ps:
        p.grad = rng.standard_normal(p.shape).astype(np.float32)
    opt = optim.AdamW(ps, lr=0.1)
    before = [np.array(host_of(p)) for p in ps]
    codes, bad.codes = bad.codes, bad.codes.cpu()
    with pytest.raises(ValueError):
        opt.step()
    bad.codes = codes
    ps[4].grad = np.ones(8)
    with pytest.raises(ValueError):
        opt.step()
    assert opt.t == 0
    for p, w, m in zip(ps, before, opt.m_t):
        assert np.array_equal(host_of(p), w) and not m.any()
    ps[4].grad = None
    opt.step()
    want = OR.adamw_step(before[0], ps[0].grad, 0 * before[0], 0 * before[0], 1, 0.1)[0]
    assert opt.t == 1 and np.array_equal(host_of(ps[0]), want)


def host_of(p):
    x = p.master if isinstance(p, BlockQuantizedParameters) else p.data
    return x if isinstance(x, np.ndarray) else x.cpu().numpy()


def test_class_with_8_bit_states():
    """The class's steps are the list's, seeded by its count."""
    rng = np.random.default_rng(11)
    ws = [rng.standard_normal(s).astype(np.float32) for s in ((64, 32), (77,), (3, 50))]
    ps = [Parameters(dev(w)) for w in ws]
    opt = optim.AdamW(ps, lr=1e-2, weight_decay=0.1, state_dtype="8bit")
    plain, states = [dev(w) for w in ws], [optim.State8.zeros(w.size) for w in ws]
    for t in range(1, 4):
        grads = [torch.randn(w.shape, device="cuda") for w in ws]
        for p, g in zip(ps, grads):
            p.grad = g
        opt.step()
        optim.adamw_step(plain, grads, states, lr=1e-2, weight_decay=0.1, step=t)
        assert all(torch.equal(p.data, w) for p, w in zip(ps, plain))
    assert opt.m_t == opt.v_t == [None] * 3
    for a, b in zip(opt.states, states):
        assert torch.equal(a.v, b.v) and torch.equal(a.m.view(torch.uint8), b.m.view(torch.uint8))
        assert torch.equal(a.m_exponents, b.m_exponents)
        assert torch.equal(a.v_exponents, b.v_exponents)


def test_refusals():
    w, g, m, v = (torch.zeros(64, device="cuda") for _ in range(4))

    def step(w=w, g=g, s=(m, v), **kw):
        optim.adamw_step([w], [g], [s], **{"lr": 0.1, "step": 1, **kw})

    step()
    with pytest.raises(TypeError):
        step(w=w.double())
    with pytest.raises(TypeError):
        step(g=g.double())
    with pytest.raises(TypeError):
        step(s=(m.half(), v))
    with pytest.raises(TypeError):
        step(w=torch.zeros(64, 2, device="cuda")[:, 0])
    with pytest.raises(ValueError):
        step(w=w.cpu())
    with pytest.raises(ValueError):
        step(g=g[:10])
    with pytest.raises(ValueError):
        step(s=(m[:10], v))
    with pytest.raises(ValueError):
        step(s=optim.State8.zeros(65))
    with pytest.raises(ValueError):
        step(step=0)
    with pytest.raises(ValueError):
        optim.adamw_step([w], [g, g], [(m, v)], lr=0.1, step=1)
    with pytest.raises(ValueError):
        optim.adamw_step([w], [g], [(m, v)], lr=0.1, step=1, decay=[True, False])
    with pytest.raises(ValueError):
        optim.adamw_step([w, w], [g, g], [(m, v), (m.clone(), v.clone())], lr=0.1, step=1)
    with pytest.raises(ValueError):
        step(s=(m, m))
    with pytest.raises(ValueError):
        step(g=m)
    step(g=w)  # (in place: the weight as its own gradient)
    with pytest.raises(ValueError):
        step(w=BlockQuantizedParameters.from_float(np.ones((8, 8), np.float32)))
    with pytest.raises(ValueError):
        optim.AdamW([Parameters(w)], lr=0.1, state_dtype="int8")
    s = optim.State8.zeros(64)
    with pytest.raises(TypeError):
        optim.State8(s.m, s.m_exponents, s.v.int(), s.v_exponents).decode()
    with pytest.raises(TypeError):
        s.decode("e4m3")


def test_a_weight_whose_scale_is_on_the_host():
    """The products move such a scale to the device; so does the step, which writes it."""
    rng = np.random.default_rng(12)
    w = (rng.standard_normal((30, 40)) * 0.05).astype(np.float32)
    a, b = (QuantizedParameters.from_float(w, "e4m3", keep_master=True) for _ in range(2))
    pair = torch.cat([b.amax, b.scale]).cpu()
    b.amax, b.scale = pair[:1], pair[1:]
    before, g = pair.clone(), torch.randn(30, 40, device="cuda")
    for p in (a, b):
        optim.adamw_step([p], [g], [tuple(torch.zeros(30, 40, device="cuda") for _ in range(2))],
                         lr=0.1, step=1)
    assert torch.equal(a.master, b.master) and torch.equal(a.scale, b.scale) and b.scale.is_cuda
    assert torch.equal(a.codes.view(torch.uint8), b.codes.view(torch.uint8))
    assert torch.equal(pair, before)


def test_captured_and_on_another_stream():
    """A captured step replayed beside eager ones: the same states and bits."""
    rng = np.random.default_rng(10)
    host = [start(rng, n, "bf16") for n in (1000, 77, 4096)]

    def fresh():
        return ([dev(h[0]) for h in host], [optim.State8.zeros(len(h[0])) for h in host])

    grads = [h[1].cuda() for h in host]
    (w, s), (w2, s2) = fresh(), fresh()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        optim.adamw_step(w, grads, s, step=1, seed=1, **HP)
    side.synchronize()
    optim.adamw_step(w2, grads, s2, step=1, seed=1, **HP)
    assert all(torch.equal(a, b) for a, b in zip(w, w2))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        optim.adamw_step(w, grads, s, step=2, seed=2, **HP)
    for _ in range(3):
        for g in grads:
            g.copy_(torch.randn_like(g))
        graph.replay()
        torch.cuda.synchronize()
        optim.adamw_step(w2, grads, s2, step=2, seed=2, **HP)
        assert all(torch.equal(a, b) for a, b in zip(w, w2))
        assert all(torch.equal(a.v, b.v) for a, b in zip(s, s2))
