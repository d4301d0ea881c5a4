"""optim's host side without a GPU: its tensors lie in host memory, and the C calls are
restated over the addresses that they are given (oracle/optim_ref.py has the step)."""
import ctypes

import numpy as np
import pytest
import torch

from novann_amd import _lib, optim, quant
from oracle import optim_ref as OR

WORDS = 16  # of novaq_adamw_tensor
NUMPY = {0: np.float32, 1: np.float16, 2: np.uint16}


def array(address, n, dtype):
    """The n values at an address, as they lie there."""
    raw = (ctypes.c_uint8 * (n * np.dtype(dtype).itemsize)).from_address(address)
    return np.frombuffer(raw, dtype)


class Library:
    """What stands for the library: fp32 states alone, and no codes."""

    def __init__(self):
        self.calls = []   # (tensors, key) of each step of many
        self.owned = {}   # address -> bytes, where a test gives them

    def novaq_status_string(self, status):
        return b"status %d" % status

    def novaq_last_hip_error(self):
        return 0

    def rows(self, table, count):
        return np.array(array(table, count * WORDS, np.int64)).reshape(count, WORDS)

    def novaq_adamw_many(self, table, count, hp, key, stream):
        rows = self.rows(table, count)
        spans = []
        for r in rows:
            n, wide = int(r[6]), 1 if r[4] else 4
            spans += [(r[0], r[0] + 4 * n, True), (r[2], r[2] + wide * n, True),
                      (r[3], r[3] + wide * n, True)]
            if r[1] != r[0]:
                spans.append((r[1], r[1] + (4 if r[7] & 0xFF == 0 else 2) * n, False))
        spans = sorted(s for s in spans if s[1] > s[0])
        last = written = 0
        for a, b, w in spans:
            if a < (last if w else written):
                return _lib.EINVAL
            last, written = max(last, b), max(written, b) if w else written
        self.calls.append((count, key))
        hp = hp._obj
        for r in rows:
            n = int(r[6])
            if r[4]:  # (states in 8 bits: the order and keys of calls are what is looked at)
                continue
            w, m, v = (array(int(r[k]), n, np.float32) for k in (0, 2, 3))
            g = array(int(r[1]), n, NUMPY[int(r[7]) & 0xFF]).astype(np.float32)
            w[...], m[...], v[...] = OR.adamw_step(
                w.copy(), g, m.copy(), v.copy(), hp.step, hp.lr, hp.beta1, hp.beta2, hp.eps,
                hp.weight_decay, bool(int(r[7]) >> 32))
        return _lib.OK

    def novaq_adamw_step_f64(self, w, g, g32, m, v, n, hp, stream):
        for at in (w, m, v):
            assert self.owned.get(at, 8 * n) >= 8 * n, "a float64 step past the end of its tensor"
        hp = hp._obj
        w, m, v = (array(at, n, np.float64) for at in (w, m, v))
        g = array(g, n, np.float32 if g32 else np.float64)
        w[...], m[...], v[...] = OR.adamw_step_f64(
            w.copy(), g.copy(), m.copy(), v.copy(), hp.step, hp.lr, hp.beta1, hp.beta2, hp.eps,
            hp.weight_decay, bool(hp.decay))
        return _lib.OK


@pytest.fixture
def library(monkeypatch):
    lib = Library()
    monkeypatch.setattr(_lib, "load", lambda: lib)
    monkeypatch.setattr(optim, "_device", lambda: torch.device("cpu"))
    monkeypatch.setattr(optim, "_get_device", lambda t: 0)
    monkeypatch.setattr(quant, "on_device", lambda dev, fn, *args: fn(*args, None))
    return lib
