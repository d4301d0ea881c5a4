"""AdamW's host side (tests/optim_host.py): which tensors its calls are given, in which order."""
import numpy as np
import pytest
import torch

from novann_amd import optim
from novann_amd.module import BlockQuantizedParameters, Parameters, QuantizedParameters
from oracle import optim_ref as OR
from tests.optim_host import library  # noqa: F401  (a fixture)

HP = dict(lr=0.01, weight_decay=0.1)


def reference(w, g, m, v, t):
    step = OR.adamw_step if w.dtype == np.float32 else OR.adamw_step_f64
    return step(w, g, m, v, t, 0.01, 0.9, 0.999, 1e-8, 0.1)


@pytest.mark.parametrize("first,later", [(np.float32, np.float64), (np.float64, np.float32)])
def test_an_array_of_another_type_steps_in_the_states_type(library, first, later):
    """.data is an attribute that a program may set: the step's type is the one that its
    states have, and an array of another is converted, both ways."""
    rng = np.random.default_rng(1)
    p = Parameters(rng.standard_normal((3, 40)).astype(first))
    opt = optim.AdamW([p], **HP)
    library.owned = {t.data_ptr(): t.numel() * t.element_size()
                     for t in (*opt._w, *opt.m_t, *opt.v_t)}
    m = v = np.zeros((3, 40), first)
    for t in (1, 2):
        w = p.data = rng.standard_normal((3, 40)).astype(later)
        p.grad = rng.standard_normal((3, 40)).astype(np.float32)
        want, m, v = reference(w.astype(first), p.grad, m, v, t)
        opt.step()
        assert p.data is w and w.dtype == later and np.array_equal(w, want.astype(later))


def test_a_scale_elsewhere_is_not_written(monkeypatch):
    """A per-tensor weight whose amax and scale lie side by side on another device than its
    master: the step has two floats of its own beside the master."""
    st, elsewhere, master = torch.ones(2), torch.ones(2), torch.zeros(4)
    place = {st.data_ptr(): 0, elsewhere.data_ptr(): -1, master.data_ptr(): 0}
    monkeypatch.setattr(optim, "_get_device", lambda t: place[t.data_ptr() & ~7])
    for pair, own in ((st, True), (elsewhere, False)):
        w = QuantizedParameters(torch.zeros(4, dtype=torch.uint8), (4,), "e4m3", pair[1:], pair[:1],
                                master=master)
        got = optim._scales(w, master)
        assert got.numel() == 2 and got.device == master.device
        assert (got.data_ptr() == pair.data_ptr()) == own


def views(kind):
    """(the buffer, parts of it that share elements, others among them that do not)."""
    base = np.random.default_rng(2).standard_normal(600).astype(np.float32)
    return base, {
        "ends": [base[:100], base[400:500], base[50:150], base[120:220]],
        "shifted by one": [base, base[1:]],
        "one inside another": [base[100:200], base[:300], base[120:130]],
        "columns and rows": [base.reshape(20, 30)[:, :7], base.reshape(20, 30)[3], base[590:]],
        "backwards": [base[300::-1], base[290:320]],
        "the same twice": [base[:50], base[50:100], base[:50]],
    }[kind]


@pytest.mark.parametrize("kind", ["ends", "shifted by one", "one inside another",
                                  "columns and rows", "backwards", "the same twice"])
def test_overlapping_arrays_step_one_after_another(library, kind):
    """As the reference steps them: each from what the one before it has left."""
    base, parts = views(kind)
    want = base.copy()

    def in_copy(a):
        at = a.__array_interface__["data"][0] - base.__array_interface__["data"][0]
        return np.ndarray(a.shape, a.dtype, want.data, at, a.strides)

    ps = [Parameters(a) for a in parts]
    opt = optim.AdamW(ps, **HP)
    rng = np.random.default_rng(3)
    states = [(np.zeros(a.shape, np.float32),) * 2 for a in parts]
    for t in (1, 2):
        for k, p in enumerate(ps):
            p.grad = rng.standard_normal(p.shape).astype(np.float32)
            w = in_copy(parts[k])
            w[...], *states[k] = reference(w.copy(), p.grad, *states[k], t)
        opt.step()
        assert np.array_equal(base, want)


def test_arrays_side_by_side_are_one_call(library):
    base = np.ones(300, np.float32)
    ps = [Parameters(base[100 * i:100 * i + 100]) for i in (2, 0, 1)] + [
        Parameters(np.ones(0, np.float32)) for _ in range(2)]
    for p in ps:
        p.grad = np.ones(p.shape, np.float32)
    optim.AdamW(ps, **HP).step()
    assert [count for count, _ in library.calls] == [5]


def block_weight():
    """Its codes and exponents on the host, where no step can write them."""
    return BlockQuantizedParameters(
        torch.zeros(8, 128, dtype=torch.uint8).view(torch.float8_e4m3fn),
        torch.zeros(1, 4, dtype=torch.uint8), (8, 16), master=torch.zeros(8, 16))


@pytest.mark.parametrize("shared", [False, True])
def test_a_step_that_is_refused_changes_nothing(library, shared):
    """One wrong parameter, in the first call or a later one: no other is stepped, and the step
    is not counted."""
    rng = np.random.default_rng(4)
    base = rng.standard_normal(100).astype(np.float32)
    wide = Parameters(rng.standard_normal(7))
    bad = block_weight()
    ps = [Parameters(base), wide, bad, Parameters(base if shared else base.copy())]
    kept = [p.data.copy() for p in (ps[0], wide, ps[3])]
    opt = optim.AdamW(ps, **HP)
    for p in ps:
        p.grad = rng.standard_normal(p.shape).astype(np.float32)
    with pytest.raises(ValueError):
        opt.step()
    wide.grad = np.ones(8)
    bad.grad = None
    with pytest.raises(ValueError):
        opt.step()
    assert opt.t == 0 and not library.calls
    for p, before in zip((ps[0], wide, ps[3]), kept):
        assert np.array_equal(p.data, before)
    assert not any(m.any() for m in opt.m_t)
    wide.grad = np.ones(7)
    want, m, _ = reference(base, ps[0].grad, 0 * base, 0 * base, 1)
    opt.step()
    assert opt.t == 1 and np.array_equal(opt.m_t[0].numpy(), m)
    assert shared or np.array_equal(ps[0].data, want)


def test_an_array_that_does_not_fit_is_refused_before_the_step(library):
    """Set to another size, to a read-only array, or (float64) to a tensor, the last of three."""
    for made, bad in ((np.float32, np.ones(5, np.float32)), (np.float64, np.ones(5)),
                      (np.float32, np.broadcast_to(np.float32(1), 6)), (np.float64, torch.ones(6))):
        ps = [Parameters(np.ones(8, np.float32)), Parameters(np.ones(8)), Parameters(np.ones(6, made))]
        opt = optim.AdamW(ps, **HP)
        for p in ps:
            p.grad = np.ones(p.shape, np.float32)
        ps[2].data = bad
        with pytest.raises((ValueError, TypeError)):
            opt.step()
        assert opt.t == 0 and (ps[0].data == 1).all() and (ps[1].data == 1).all()


def test_a_gradient_that_is_another_weight(library):
    """The weight is stepped after the parameter whose gradient it was."""
    rng = np.random.default_rng(5)
    a, b, c = (torch.from_numpy(rng.standard_normal(60).astype(np.float32)) for _ in range(3))
    ps = [Parameters(a), Parameters(b), Parameters(c)]
    ps[0].grad, ps[1].grad, ps[2].grad = b, torch.ones(60), torch.ones(60)
    zero = np.zeros(60, np.float32)
    want = [reference(x.numpy().copy(), g.numpy().copy(), zero, zero, 1)[0]
            for x, g in ((a, b), (b, torch.ones(60)), (c, torch.ones(60)))]
    optim.AdamW(ps, **HP).step()
    assert [count for count, _ in library.calls] == [2, 1]
    for x, w in zip((a, b, c), want):
        assert np.array_equal(x.numpy(), w)


def test_each_call_has_random_numbers_of_its_own(library):
    """States in 8 bits of parameters that take turns: every call counts its elements from the
    list's first, so no two calls may have one key, in a step or in the next ones."""
    base = np.ones(200, np.float32)
    w = torch.ones(64)
    ps = [Parameters(base), Parameters(base[100:]), Parameters(base[150:]), Parameters(w),
          Parameters(torch.ones(64))]
    opt = optim.AdamW(ps, state_dtype="8bit", **HP)
    for p in ps:
        p.grad = torch.ones(p.shape)
    ps[4].grad = w  # (its turn is after w's)
    for _ in range(3):
        opt.step()
    keys = [key for _, key in library.calls]
    assert len(keys) >= 9 and len(set(keys)) == len(keys)
    # the first call's is the step's own
    assert library.calls[0][1] == optim._key(1)


def test_the_moments_that_are_set_are_the_ones_that_step(library):
    """m_t and v_t are the optimizer's state: what a program puts there, as it does when it goes
    on from a checkpoint, is what the next step reads."""
    rng = np.random.default_rng(6)
    ps = [Parameters(rng.standard_normal(20).astype(np.float32)),
          Parameters(rng.standard_normal(20))]
    opt = optim.AdamW(ps, **HP)
    assert type(opt.m_t) is type(opt.v_t) is list
    for way in range(3):
        m, v = ([abs(rng.standard_normal(20)).astype(p.data.dtype) for p in ps] for _ in range(2))
        new = [[torch.from_numpy(a.copy()) for a in x] for x in (m, v)]
        if way == 0:
            opt.m_t, opt.v_t = new
        elif way == 1:
            for i in range(2):
                opt.m_t[i], opt.v_t[i] = new[0][i], new[1][i]
        else:
            opt.states = list(zip(*new))
        assert all(opt.states[i][0] is opt.m_t[i] is new[0][i] for i in range(2))
        want = []
        for p, a, b in zip(ps, m, v):
            p.grad = rng.standard_normal(20).astype(np.float32)
            want.append(reference(p.data.copy(), p.grad, a, b, way + 1))
        opt.step()
        for i, (p, (w, a, b)) in enumerate(zip(ps, want)):
            assert np.array_equal(p.data, w)
            assert np.array_equal(opt.m_t[i].numpy(), a) and np.array_equal(opt.v_t[i].numpy(), b)
    opt.m_t[1] = torch.zeros(20)  # (float32 beside a float64 parameter)
    with pytest.raises(ValueError):
        opt.step()
    opt.m_t[1] = torch.zeros(20, dtype=torch.float64)
    opt.m_t[0] = torch.zeros(19)
    with pytest.raises(ValueError):
        opt.step()
    assert opt.t == 3


def test_states_in_8_bits_are_set_as_a_whole(library):
    p = Parameters(torch.zeros(300))
    p.grad = torch.ones(300)
    opt = optim.AdamW([p], state_dtype="8bit", **HP)
    assert opt.m_t == opt.v_t == [None] and isinstance(opt.states[0], optim.State8)
    new = optim.State8.zeros(300)
    opt.states[0] = tuple(new)
    assert opt.states[0] == new and opt.states[-1:] == [new]
    opt.step()
    with pytest.raises(ValueError):
        opt.states = []
    opt.states = [(torch.zeros(300), torch.zeros(300))]
    opt.step()
    assert opt.m_t[0].any()


@pytest.mark.parametrize("n", [0, 1, 126, 127, 129, 1000, 2049])
def test_new_states_are_aligned(n):
    """All four on 16 bytes, whatever the size: one tensor that is not makes its whole step go
    an element at a time."""
    s = optim.State8.zeros(n, torch.device("cpu"))
    for t, k in zip(s, (n, -(-n // 128)) * 2):
        assert t.numel() == k and t.is_contiguous() and t.data_ptr() % 16 == 0
        assert not t.view(torch.uint8).any()
