"""Plain 64-bit forms of the token operators (numpy), and random tables of
every stored type, shared by their tests."""
from __future__ import annotations

import numpy as np
import torch

from novann_amd.module import Parameters, QuantizedParameters

TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
# half an ulp, relative: the largest error of one rounding to nearest of p bits
# is 2^-p (p = 24, 8 and 11)
HALF_ULP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
# half the smallest subnormal: what a rounding may be off where values are small
HALF_MIN = {"f32": 2.0 ** -150, "bf16": 2.0 ** -134, "f16": 2.0 ** -25}


def table(rng, V, D, dtype, std=1.0):
    """(weight as the operators take it, its values in float64)."""
    w = (rng.standard_normal((V, D)) * std).astype(np.float32)
    if dtype in ("e4m3", "e5m2", "e2m1"):
        q = QuantizedParameters.from_float(w, dtype)
        return q, dense(q)
    t = torch.from_numpy(w).cuda().to(TORCH[dtype])
    return Parameters(t), t.double().cpu().numpy()


def dense(q):
    """dec(codes) * s in float64 (codes decoded exactly, one fp32 scale)."""
    one = QuantizedParameters(q.codes, q.shape, q.dtype, torch.ones_like(q.scale))
    return one.dequantize().double().cpu().numpy() * float(q.scale)


def floats(rng, shape, dtype, std=1.0):
    t = torch.from_numpy((rng.standard_normal(shape) * std).astype(np.float32)).cuda()
    return t.to(TORCH[dtype])


def host(t):
    return t.double().cpu().numpy()


def cross_entropy(x, w, t, ignore=-100):
    """(loss of each row, lse, softmax) of float64 x (N, D), w (V, D)."""
    l = x @ w.T
    top = l.max(1, keepdims=True)
    e = np.exp(l - top)
    lse = np.log(e.sum(1)) + top[:, 0]
    kept = t != ignore
    at = np.where(kept, t, 0)
    each = np.where(kept, lse - l[np.arange(len(t)), at], 0.0)
    return each, lse, e / e.sum(1, keepdims=True)


def cross_entropy_grads(x, w, t, f, ignore=-100):
    """(P, grad_x, grad_w) for the row gradients f (float64)."""
    _, _, p = cross_entropy(x, w, t, ignore)
    kept = t != ignore
    p[np.arange(len(t))[kept], t[kept]] -= 1.0
    p *= np.where(kept, f, 0.0)[:, None]
    p[~kept] = 0.0
    xs = np.where(kept[:, None], x, 0.0)
    return p, p @ w, p.T @ xs
