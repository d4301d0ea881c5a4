"""AdamW with NovaNN's interface (novann/optim/adamw.py:6-69), on the GPU.

Same constructor (parameters, lr, betas, weight_decay, epsilon), ``step`` and
``zero_grad``; BatchNorm gamma / beta (by name) are not decayed, as there.  All
parameters with a gradient step in one call over the list (``adamw_step``,
libnovaq ``novaq_adamw_many``), those that share memory in calls one after
another; their states are in fp32 or in 8 bits.  With fp32 states each element
takes the float32 update the reference computes on its float32 arrays, bit for
bit.  ``QuantizedParameters`` and ``BlockQuantizedParameters`` step their fp32
``master`` weights, and their codes and scales are written again in the same
call.  ``Parameters`` holding numpy arrays are uploaded at every step (so changes
a caller makes to ``.data`` between steps count, as with the reference), stepped
on the device and written back in place.  float64 arrays (the BatchNorm gamma /
beta, float64 in the reference too) keep float64 moments and step in float64 with
numpy's promotion of a float32 gradient (``novaq_adamw_step_f64``); any other
numpy array steps in float32 (the reference's float32 parameters).
"""
from __future__ import annotations

import ctypes
import itertools
import math
from array import array
from collections.abc import Sequence
from operator import attrgetter
from typing import Iterable, List, NamedTuple, Optional

import numpy as np
import torch

from . import _lib, quant
from ._lib import DTYPES, check
from .module import BlockQuantizedParameters, Parameters, QuantizedParameters


# (steps and clipping handle hundreds of tensors a call: whole lists at a time, a
# few tenths of a microsecond a tensor)
_data_ptr, _numel = torch.Tensor.data_ptr, torch.Tensor.numel
_contiguous, _get_device = torch.Tensor.is_contiguous, torch.Tensor.get_device
_dtype, _is_cuda = attrgetter("dtype"), attrgetter("is_cuda")


def _device() -> torch.device:
    if not torch.cuda.is_available():
        raise RuntimeError("novann_amd needs a HIP device (no CPU fallback)")
    return torch.device("cuda", torch.cuda.current_device())


def _dev_f32(a, dev) -> torch.Tensor:
    if isinstance(a, np.ndarray):
        return torch.from_numpy(np.ascontiguousarray(a, dtype=np.float32)).to(dev)
    return a.to(device=dev, dtype=torch.float32).contiguous()


def _is_f64(p) -> bool:
    d = getattr(p, "data", None)
    return isinstance(d, np.ndarray) and d.dtype == np.float64


def _dev_grad64(g, dev):
    """A float64 parameter's gradient on the device in the dtype numpy would
    compute with: float32 stays float32, anything else becomes float64."""
    if isinstance(g, torch.Tensor):
        g = g.detach().cpu().numpy()
    g = np.asarray(g)
    dt = np.float32 if g.dtype == np.float32 else np.float64
    return torch.from_numpy(np.ascontiguousarray(g, dtype=dt)).to(dev), dt == np.float32


class State8(NamedTuple):
    """AdamW's two states of n elements in 8 bits, 128 in a row sharing an exponent each.

    m: E4M3 codes (n), m_exponents: uint8 (ceil(n / 128)), a scale of 2^(e - 127); v: uint8
    codes (n) without a sign, 5 bits of exponent and 3 of mantissa (c > 0 is the float with
    the bits (c << 20) + ((e - 31) << 23)), v_exponents as m's.  A step rounds both at
    random (see ``adamw_step``)."""

    m: torch.Tensor
    m_exponents: torch.Tensor
    v: torch.Tensor
    v_exponents: torch.Tensor

    @classmethod
    def zeros(cls, n: int, device=None) -> "State8":
        dev, blocks = device or _device(), -(-n // quant.BLOCK)
        # (rows of whole 16 bytes: a step whose tensors are aligned takes four elements at a time)
        codes, exponents = (torch.zeros(2, -(-k // 16) * 16, dtype=torch.uint8, device=dev)[:, :k]
                            for k in (n, blocks))
        return cls(codes[0].view(torch.float8_e4m3fn), exponents[0], codes[1], exponents[1])

    def check(self, what: str = "state") -> None:
        n = self.m.numel()
        if self.m.dtype is not torch.float8_e4m3fn or self.v.dtype is not torch.uint8 or \
                self.m_exponents.dtype is not torch.uint8 or \
                self.v_exponents.dtype is not torch.uint8:
            raise TypeError(f"{what}: m is float8_e4m3fn, v and the exponents uint8")
        blocks = -(-n // quant.BLOCK)
        if self.v.numel() != n or self.m_exponents.numel() != blocks or \
                self.v_exponents.numel() != blocks:
            raise ValueError(f"{what}: {n} elements have as many codes and {blocks} exponents each")
        for t in (self.m, self.v, self.m_exponents, self.v_exponents):
            if not t.is_contiguous() or t.device != self.m.device or not t.is_cuda:
                raise ValueError(f"{what}: codes and exponents must be contiguous, on one CUDA "
                                 "(HIP) device")

    def decode(self, dtype: str = "f32"):
        """(m, v) in 'f32', 'bf16' (both exact) or 'f16', of m's shape."""
        self.check()
        if dtype not in ("f32", "bf16", "f16"):
            raise TypeError(f"states decode to f32, bf16 or f16, got {dtype!r}")
        m = torch.empty(self.m.shape, dtype=quant.STORAGE[dtype], device=self.m.device)
        v = torch.empty_like(m)
        check(quant.on_device(
            m.device, _lib.load().novaq_adamw_state_decode, self.m.data_ptr(),
            self.m_exponents.data_ptr(), self.v.data_ptr(), self.v_exponents.data_ptr(),
            m.numel(), m.data_ptr(), v.data_ptr(), DTYPES[dtype]), "state decode")
        return m, v


_M64 = (1 << 64) - 1


def _key(seed: int) -> int:
    """A seed's 32 bits for the rounding of states: three multiplications by the
    fractional parts of the golden ratio and of the square roots of 3 and 2, their halves
    folded, so that seeds that follow one another have nothing in common."""
    x = (int(seed) * 0x9E3779B97F4A7C15 + 0x3C6EF372FE94F82B) & _M64
    x = ((x ^ (x >> 32)) * 0xBB67AE8584CAA73B) & _M64
    x = ((x ^ (x >> 29)) * 0x6A09E667F3BCC909) & _M64
    return x >> 32


_STEP_GRADS = {torch.float32: DTYPES["f32"], torch.float16: DTYPES["f16"],
               torch.bfloat16: DTYPES["bf16"]}
_ROW = 16  # words of novaq_adamw_tensor


def _master(w):
    """The fp32 weights that a step changes."""
    if isinstance(w, (QuantizedParameters, BlockQuantizedParameters)):
        if w.master is None:
            raise ValueError(f"AdamW: {type(w).__name__} need fp32 master weights "
                             "(from_float(..., keep_master=True))")
        return w.master
    return w.data if isinstance(w, Parameters) else w


def _types(tensors, dtypes, what: str) -> list:
    """The codes of the tensors' types, which must be among dtypes (TypeError)."""
    types = list(map(_dtype, tensors))
    if types[0] in dtypes and types.count(types[0]) == len(types):  # (the ordinary list)
        return [dtypes[types[0]]] * len(types)
    codes = [dtypes.get(t) for t in types]
    if None in codes:
        raise TypeError(f"AdamW: {what} must be contiguous "
                        f"{' or '.join(str(t)[6:] for t in dtypes)}, got "
                        f"{types[codes.index(None)]}")
    return codes


def _as_many(tensors, counts, what: str) -> None:
    have = list(map(_numel, tensors))
    if have != counts:
        k = next(k for k, c in enumerate(counts) if have[k] != c)
        raise ValueError(f"AdamW: {what} of {have[k]} values for a parameter of {counts[k]}")


def _stored(table: array, at: int, w, n: int, amax_scale, dev: int) -> None:
    """The fields of a row (from word `at` on) that say what a quantized weight on device
    `dev` is stored as."""
    codes = [w.codes]
    if isinstance(w, QuantizedParameters):
        if math.prod(w.stored_shape) != n:
            raise ValueError(f"AdamW: a {w.shape} weight's master has {n} values")
        quant._require_holds(w.codes, w.dtype, n, "AdamW: weight codes")
        quant._require_device(w.codes, "AdamW: weight codes")
        table[at + 8], table[at + 12] = w.codes.data_ptr(), amax_scale.data_ptr()
    else:
        if math.prod(w.shape) != n:
            raise ValueError(f"AdamW: a {w.shape} weight's master has {n} values")
        w.blocks().check("weight")
        t = w.blocks_t()
        table[at + 8], table[at + 9] = w.codes.data_ptr(), w.exponents.data_ptr()
        if t is not None:
            t.check("transposed weight")
            table[at + 10], table[at + 11] = t.data.data_ptr(), t.exponents.data_ptr()
            codes.append(t.data)
        table[at + 13], table[at + 14] = w.shape
    if any(c.get_device() != dev for c in codes):
        raise ValueError("AdamW: a weight's codes must be on its master's device")
    table[at + 15] = DTYPES[w.dtype]


_F32, _U8, _E4M3 = {torch.float32: 0}, {torch.uint8: 0}, {torch.float8_e4m3fn: 0}
# the words of a row that a state's tensors go to
_STATES, _STATES8 = ((2, _F32), (3, _F32)), ((2, _E4M3), (4, _U8), (3, _U8), (5, _U8))


def _rows(weights, masters, grads, states, decay, scales) -> array:
    """The rows of novaq_adamw_tensor for lists of at least one, once everything that they
    name is looked at.  masters: what is stepped; decay: a list or None; scales: for each
    weight where a per-tensor one's amax and scale go, or None."""
    counts = list(map(_numel, masters))
    sizes = list(map(len, states))
    if sizes.count(2) + sizes.count(4) != len(sizes):
        raise ValueError("AdamW: a state is (m, v) or a State8")
    _types(masters, _F32, "device parameters")
    types = _types(grads, _STEP_GRADS, "gradients")
    _as_many(grads, counts, "gradient")
    if decay is None:
        types = [t | 1 << 32 for t in types]
    else:
        types = [t | bool(d) << 32 for t, d in zip(types, decay)]
    table = array("q", bytes(8 * _ROW * len(masters)))
    table[0::_ROW] = array("q", list(map(_data_ptr, masters)))
    table[1::_ROW] = array("q", list(map(_data_ptr, grads)))
    table[6::_ROW] = array("q", counts)
    table[7::_ROW] = array("q", types)
    everything = masters + grads
    for size, columns in ((2, _STATES), (4, _STATES8)):
        if size not in sizes:
            continue
        which, ours, some = None, counts, states
        if sizes.count(size) < len(sizes):
            which = [i for i, k in enumerate(sizes) if k == size]
            ours, some = [counts[i] for i in which], [states[i] for i in which]
        for (column, dtypes), tensors in zip(columns, zip(*some)):
            _types(tensors, dtypes, "states")
            _as_many(tensors, ours if column < 4 else [-(-c // quant.BLOCK) for c in ours],
                     "state")
            everything += tensors
            at = list(map(_data_ptr, tensors))
            if which is None:
                table[column::_ROW] = array("q", at)
            else:
                for i, p in zip(which, at):
                    table[column + _ROW * i] = p
    dev = _get_device(masters[0])
    if dev < 0 or set(map(_get_device, everything)) != {dev}:
        raise ValueError("AdamW: parameters, gradients and states must be CUDA (HIP) device "
                         f"tensors on one device, got {set(map(_get_device, everything))} (-1: "
                         "the host)")
    if not all(map(_contiguous, everything)):
        raise TypeError("AdamW: parameters, gradients and states must be contiguous")
    for i, w in enumerate(weights):
        if isinstance(w, (QuantizedParameters, BlockQuantizedParameters)):
            _stored(table, _ROW * i, w, counts[i], scales[i], dev)
    return table


def _launch(table: array, weights, scales, dev, hp, seed: int) -> int:
    """The C call's status; nothing was launched where it is NOVAQ_EINVAL."""
    rc = quant.on_device(dev, _lib.load().novaq_adamw_many, table.buffer_info()[0],
                         len(table) // _ROW, ctypes.byref(hp), _key(seed))
    if rc == _lib.OK:
        for w, st in zip(weights, scales):
            if st is not None:
                # the codes and scale the products read now follow the master (the next step
                # rewrites st after this step's readers, in stream order)
                w.amax, w.scale = st[0:1], st[1:2]
    return rc


def _scales(w, master) -> Optional[torch.Tensor]:
    """Two adjacent floats on the master's device for a per-tensor weight's amax and scale: its
    own where they are adjacent there, so that who reads them goes on with the new ones (a
    product moves a scale that lies elsewhere, the step writes where it says)."""
    if not isinstance(w, QuantizedParameters):
        return None
    a, s = w.amax, w.scale
    if isinstance(a, torch.Tensor) and a.dtype == s.dtype == torch.float32 and \
            _get_device(a) == _get_device(s) == _get_device(master) and \
            s.data_ptr() == a.data_ptr() + 4 and a.untyped_storage().data_ptr() == \
            s.untyped_storage().data_ptr():
        return a.as_strided((2,), (1,))
    return torch.empty(2, dtype=torch.float32, device=master.device)


def adamw_step(weights: Iterable, grads: Iterable, states: Iterable, *, lr: float, step: int,
               betas=(0.9, 0.999), weight_decay: float = 0.0, epsilon: float = 1e-8,
               decay: Optional[Iterable] = None, seed: Optional[int] = None) -> None:
    """One AdamW step (adamw.py:41-65) of many tensors in place, in one launch for 48.

    weights: fp32 device tensors or Parameters of them, QuantizedParameters or
    BlockQuantizedParameters (their masters are stepped, and their codes and scales written
    again); grads: fp32, bf16 or f16 device tensors of as many elements (None: the weight is
    passed over); states: for each weight (m, v), two fp32 tensors, or a State8 (or its
    four tensors).  ``step`` is the count t from 1 on; ``decay``: truth values, false for
    weights that are not decayed.  Tensors that share memory are a ValueError.

    With fp32 states each element takes the reference's float32 operations, bit for bit;
    beside states in 8 bits the step's root and quotient are the hardware's (2^-20 of the
    step).  States in 8 bits are rounded up with the probability of their place between two codes
    (nearest would keep a v that moves by a thousandth where it is), by random numbers
    from ``seed`` (the step count by default) and an element's place: equal calls give equal
    bits, and a captured one replays its step count and seed."""
    weights, grads, states = list(weights), list(grads), list(states)
    flags = None if decay is None else list(decay)
    if not len(weights) == len(grads) == len(states) or \
            flags is not None and len(flags) != len(weights):
        raise ValueError(f"{len(weights)} weights, {len(grads)} gradients, {len(states)} states"
                         + ("" if flags is None else f", {len(flags)} decay flags"))
    if int(step) < 1:
        raise ValueError(f"step counts from 1 on, got {step}")
    hp = _lib.AdamW(float(lr), float(betas[0]), float(betas[1]), float(epsilon),
                    float(weight_decay), int(step), 1)
    keep = [i for i, g in enumerate(grads) if g is not None]
    if not keep:
        return
    if len(keep) < len(grads):
        weights, grads, states = ([a[i] for i in keep] for a in (weights, grads, states))
        flags = None if flags is None else [flags[i] for i in keep]
    masters = weights
    if set(map(type, weights)) != {torch.Tensor}:
        masters = [_master(w) for w in weights]
    if not all(map(_contiguous, grads)):
        grads = [g.contiguous() for g in grads]
    scales = [None] * len(weights) if masters is weights else list(map(_scales, weights, masters))
    table = _rows(weights, masters, grads, states, flags, scales)
    check(_launch(table, weights, scales, masters[0].device, hp, step if seed is None else seed),
          "adamw step")


def _span(a):
    """Where the elements of an array (-1) or of a contiguous device tensor (its device's
    index) lie: (place, first byte, end)."""
    if isinstance(a, torch.Tensor):
        at = a.data_ptr()
        return _get_device(a), at, at + a.numel() * a.element_size()
    at = a.__array_interface__["data"][0]
    if a.flags.c_contiguous or a.size == 0:
        return -1, at, at + a.nbytes
    reach = [(n - 1) * s for n, s in zip(a.shape, a.strides)]
    return (-1, at + sum(r for r in reach if r < 0),
            at + sum(r for r in reach if r > 0) + a.itemsize)


def _turns(count: int, spans) -> list:
    """For each of so many parameters 0, or one more than the last turn of the earlier ones
    whose memory it shares.  spans: (parameter, place, first byte, end, whether the step writes
    there); what is only read may be shared."""
    spans = sorted((s for s in spans if s[2] < s[3]), key=lambda s: s[1:3])
    before = {}  # parameter -> the earlier ones that it waits for
    group, place, end = [], None, 0

    def share(group):
        for k, a in enumerate(group):
            for b in group[:k]:
                if a[0] != b[0] and (a[4] or b[4]) and a[2] < b[3] and b[2] < a[3]:
                    before.setdefault(max(a[0], b[0]), []).append(min(a[0], b[0]))

    # (groups of spans that reach into one another, from first bytes in order)
    for s in spans:
        if s[1] != place or s[2] >= end:
            share(group)
            group, place, end = [], s[1], 0
        group.append(s)
        end = max(end, s[3])
    share(group)
    turns = [0] * count
    for i in sorted(before):
        turns[i] = 1 + max(turns[j] for j in before[i])
    return turns


class _States(Sequence):
    """An AdamW's states, each (m_t[i], v_t[i]) or a State8, as a list that writes through."""

    def __init__(self, opt) -> None:
        self._opt = opt

    def __len__(self) -> int:
        return len(self._opt.m_t)

    def __getitem__(self, i):
        if isinstance(i, slice):
            return [self[k] for k in range(*i.indices(len(self)))]
        m, v = self._opt.m_t[i], self._opt.v_t[i]
        return self._opt._state8[i] if m is None and v is None else (m, v)

    def __setitem__(self, i: int, state) -> None:
        pair, codes = (state, None) if len(state) == 2 else ((None, None), State8(*state))
        (self._opt.m_t[i], self._opt.v_t[i]), self._opt._state8[i] = pair, codes


class AdamW:
    """AdamW with decoupled weight decay (adamw.py:6-69).

    ``state_dtype`` '8bit' keeps the moments of fp32 (master) weights as State8; float64
    parameters keep theirs in float64."""

    def __init__(self, parameters: Iterable, lr: float, betas=(0.9, 0.999),
                 weight_decay: float = 0, epsilon: float = 1e-8, state_dtype: str = "f32") -> None:
        if state_dtype not in ("f32", "8bit"):
            raise ValueError(f"state_dtype must be 'f32' or '8bit', got {state_dtype!r}")
        self.params: List = list(parameters)
        self.lr, self.wd = float(lr), float(weight_decay)
        self.b1, self.b2 = float(betas[0]), float(betas[1])
        self.eps = float(epsilon)
        self.t = 0
        dev = _device()
        self._w: List[torch.Tensor] = []
        for p in self.params:
            if isinstance(p, (QuantizedParameters, BlockQuantizedParameters)):
                self._w.append(_master(p))
            elif _is_f64(p):
                self._w.append(torch.from_numpy(np.ascontiguousarray(p.data)).to(dev))
            elif isinstance(p.data, np.ndarray):
                self._w.append(_dev_f32(p.data, dev))
            else:
                if p.data.dtype != torch.float32 or not p.data.is_contiguous():
                    raise TypeError("AdamW: device parameters must be contiguous float32")
                self._w.append(p.data)
        self._state8 = [State8.zeros(w.numel(), w.device)
                        if state_dtype == "8bit" and w.dtype == torch.float32 else None
                        for w in self._w]
        # the moments that the next step reads, None where they are in 8 bits
        self.m_t, self.v_t = ([torch.zeros_like(w) if s is None else None
                               for w, s in zip(self._w, self._state8)] for _ in range(2))
        self._amax_scale: List[Optional[torch.Tensor]] = [
            torch.empty(2, dtype=torch.float32, device=w.device)
            if isinstance(p, QuantizedParameters) else None for p, w in zip(self.params, self._w)]

    @property
    def states(self) -> _States:
        """Each parameter's (m_t[i], v_t[i]), or its State8."""
        return _States(self)

    @states.setter
    def states(self, states) -> None:
        states = list(states)
        if len(states) != len(self.params):
            raise ValueError(f"{len(states)} states for {len(self.params)} parameters")
        for i, state in enumerate(states):
            self.states[i] = state

    def _grad(self, p, w: torch.Tensor) -> torch.Tensor:
        """A parameter's gradient as the step reads it."""
        g = p.grad
        if type(g) is torch.Tensor and g.dtype in _STEP_GRADS and g.shape == w.shape and \
                _get_device(g) == _get_device(w) and g.is_contiguous():
            return g
        if not (isinstance(g, torch.Tensor) and g.device == w.device and g.dtype in _STEP_GRADS):
            g = _dev_f32(g, w.device)
        if isinstance(p, QuantizedParameters) and p.stored_shape != p.shape:
            # the pad column of an odd-width E2M1 weight: zero gradient
            g = torch.nn.functional.pad(g.reshape(p.shape), (0, 1))
        return g.contiguous().reshape(w.shape)

    def _hp(self, decay: int, t: int) -> "_lib.AdamW":
        return _lib.AdamW(self.lr, self.b1, self.b2, self.eps, self.wd, t, decay)

    def step(self) -> None:
        """One optimization step (adamw.py:41-65).  All gradients, states and codes are looked
        at before anything is launched: a step that is refused changes nothing."""
        t = self.t + 1
        wide, listed, grads = [], [], {}
        for i, p in enumerate(self.params):
            if p.grad is None:
                continue
            self._array(i)
            if self._w[i].dtype == torch.float64:  # (its states' type, whatever .data is now)
                wide.append((i, *self._grad64(i)))
            else:
                listed.append(i)
                grads[i] = self._grad(p, self._w[i])
        calls = self._calls(listed) if listed else []
        tables = [self._rows(call, grads) for call in calls]
        # (each call's random numbers are its own: seeds past any step count)
        seeds = itertools.count(t, 1 << 32)
        for call, table in zip(calls, tables):
            self._step_call(call, table, grads, t, seeds)
            self.t = t
        for i, g, g32 in wide:
            self._step_f64(i, g, g32, t)
            self.t = t
        self.t = t

    def _calls(self, listed: List[int]) -> List[List[int]]:
        """The parameters by call.  Those that share memory (a weight named twice, views of one
        buffer) step one after another, in their order: an array's bytes are its own, its device
        copy is not.  (Device tensors that overlap but start apart are found by the C call.)"""
        ws = [self._w[i] for i in listed]
        arrays = [i for i in listed if isinstance(getattr(self.params[i], "data", None), np.ndarray)]
        if len(arrays) < 2 and len(set(map(_data_ptr, ws))) == len(ws) == \
                list(map(_get_device, ws)).count(_get_device(ws[0])):
            return [listed]
        arrays = set(arrays)
        turns = _turns(len(listed), [
            (k, *_span(self.params[i].data if i in arrays else w), True)
            for k, (i, w) in enumerate(zip(listed, ws))])
        calls = {}
        for turn, i in sorted(zip(turns, listed)):
            calls.setdefault((turn, self._w[i].device), []).append(i)
        return list(calls.values())

    def _rows(self, call: List[int], grads) -> array:
        ps, states = [self.params[i] for i in call], self.states
        return _rows(ps, [self._w[i] for i in call], [grads[i] for i in call],
                     [states[i] for i in call],
                     [getattr(p, "name", None) not in ("gamma", "beta") for p in ps],
                     [self._amax_scale[i] for i in call])

    def _launch(self, call: List[int], table: array, t: int, seed: int) -> int:
        return _launch(table, [self.params[i] for i in call], [self._amax_scale[i] for i in call],
                       self._w[call[0]].device, self._hp(1, t), seed)

    def _memory(self, k: int, i: int, g: torch.Tensor):
        """The spans of parameter i of a call, its k-th."""
        p, w = self.params[i], self._w[i]
        written = [w, *self.states[i], self._amax_scale[i]]
        written += [getattr(p, name, None) for name in ("codes", "exponents", "codes_t",
                                                        "exponents_t")]
        spans = [(k, *_span(x), True) for x in written if x is not None]
        if g.data_ptr() != w.data_ptr():
            spans.append((k, *_span(g), False))
        return spans

    def _step_call(self, call: List[int], table: array, grads, t: int, seeds) -> None:
        arrays = [(p.data, self._w[i]) for i, p in ((i, self.params[i]) for i in call)
                  if isinstance(getattr(p, "data", None), np.ndarray)]
        for data, w in arrays:
            # the caller may have changed .data since the last step
            w.copy_(torch.from_numpy(np.ascontiguousarray(data).reshape(w.shape).astype(
                np.float32, copy=False)))
        seed = next(seeds)
        rc = self._launch(call, table, t, seed)
        if rc == _lib.EINVAL:
            # memory that parameters share otherwise (one's gradient another's weight): in turn too
            turns = _turns(len(call), [s for k, i in enumerate(call)
                                       for s in self._memory(k, i, grads[i])])
            for turn in range(max(turns) + 1) if any(turns) else ():
                part = [i for i, n in zip(call, turns) if n == turn]
                rc = self._launch(part, self._rows(part, grads), t, seed if turn == 0 else next(seeds))
                check(rc, "adamw step")
        check(rc, "adamw step")
        for data, w in arrays:
            data[...] = w.cpu().numpy().reshape(data.shape)

    def _array(self, i: int) -> None:
        """A parameter's .data, where it is an array: the step reads and writes it."""
        data, w = getattr(self.params[i], "data", None), self._w[i]
        if isinstance(data, np.ndarray):
            if data.size != w.numel():
                raise ValueError(f"AdamW: an array of {data.size} values for a parameter of {w.numel()}")
            if not data.flags.writeable:
                raise ValueError("AdamW: a parameter's array is read-only")
        elif w.dtype == torch.float64:
            raise TypeError("AdamW: a float64 parameter is a numpy array")

    def _grad64(self, i: int):
        w = self._w[i]
        g, g32 = _dev_grad64(self.params[i].grad, w.device)
        if g.numel() != w.numel():
            raise ValueError(f"AdamW: gradient of {g.numel()} values for a parameter of {w.numel()}")
        for s in (self.m_t[i], self.v_t[i]):
            if s.dtype != torch.float64 or s.numel() != w.numel() or not s.is_contiguous() or \
                    _get_device(s) != _get_device(w):
                raise ValueError("AdamW: a float64 parameter's states are contiguous float64 tensors "
                                 "of as many elements, beside it")
        return g, g32

    def _step_f64(self, i: int, g: torch.Tensor, g32: bool, t: int) -> None:
        p, w = self.params[i], self._w[i]
        w.copy_(torch.from_numpy(np.ascontiguousarray(p.data, dtype=np.float64).reshape(w.shape)))
        hp = self._hp(0 if getattr(p, "name", None) in ("gamma", "beta") else 1, t)
        check(quant.on_device(w.device, _lib.load().novaq_adamw_step_f64, w.data_ptr(), g.data_ptr(),
                              int(g32), self.m_t[i].data_ptr(), self.v_t[i].data_ptr(), w.numel(),
                              ctypes.byref(hp)), "adamw f64")
        p.data[...] = w.cpu().numpy().reshape(p.data.shape)

    def zero_grad(self, set_to_none: bool = False) -> None:
        """Clears the gradients of all optimized parameters (adamw.py:67-70)."""
        for p in self.params:
            p.zero_grad(set_to_none=set_to_none)


_GRAD_TYPES = {torch.float32: DTYPES["f32"], torch.float16: DTYPES["f16"],
               torch.bfloat16: DTYPES["bf16"], torch.float64: _lib.F64}


def _type_codes(tensors, what: str) -> list:
    """The type codes of device tensors that may be clipped (else TypeError or
    ValueError)."""
    types = list(map(_dtype, tensors))
    if types and types.count(types[0]) == len(types):  # (the ordinary list)
        codes = [_GRAD_TYPES.get(types[0])] * len(types)
    else:
        codes = list(map(_GRAD_TYPES.get, types))
    if None in codes:
        raise TypeError(f"{what} must be fp32, f16, bf16 or float64, got "
                        f"{types[codes.index(None)]}")
    if not all(map(_is_cuda, tensors)):
        raise ValueError(f"{what} must be CUDA (HIP) device tensors, got one on the host")
    return codes


def _clip(grads, at, outs, max_norm: float, eps: float) -> torch.Tensor:
    """The C call on contiguous device tensors; at: their addresses; outs: where the
    clipped ones go, or None."""
    n = len(grads)
    dev = grads[0].device if n else _device()
    # the rows of novaq_gradient: address, address, count, the two types (an array
    # is made of a list in less time than of an iterator)
    types = _type_codes(grads, "gradients")
    counts = list(map(_numel, grads))
    table = array("q", bytes(32 * n))
    table[0::4] = at = array("q", at)
    table[2::4] = array("q", counts)
    if outs is not None:
        if outs is not grads and list(map(_numel, outs)) != counts:
            raise ValueError("every out must have as many elements as its gradient")
        to = types if outs is grads else _type_codes(outs, "out")
        types = [a | b << 32 for a, b in zip(types, to)]
        table[1::4] = at if outs is grads else array("q", list(map(_data_ptr, outs)))
    table[3::4] = array("q", types)
    lib = _lib.load()
    nbytes = lib.novaq_clip_grad_norm_workspace(n)
    work = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    norm = torch.empty((), dtype=torch.float32, device=dev)
    check(lib.novaq_clip_grad_norm(table.buffer_info()[0] if n else None, n, max_norm, eps,
                                   norm.data_ptr(), work.data_ptr(), nbytes,
                                   torch._C._cuda_getCurrentRawStream(dev.index)),
          "clip_grad_norm")
    return norm


def _elements(g):
    """The memory that a gradient's elements lie in: address, type and layout."""
    if isinstance(g, np.ndarray):
        whole, at = g.flags.c_contiguous, g.__array_interface__["data"][0]
        return at, g.dtype, g.size if whole else (g.shape, g.strides)
    return g.data_ptr(), g.dtype, g.numel() if g.is_contiguous() else (g.shape, g.stride())


def _distinct(grads) -> list:
    """The gradients, one whose elements an earlier one names left out: it would
    count twice, and be scaled twice in place."""
    kept, seen = [], set()
    for g in grads:
        if isinstance(g, (torch.Tensor, np.ndarray)) and math.prod(g.shape) > 0:
            at = _elements(g)
            if at in seen:
                continue
            seen.add(at)
        kept.append(g)
    return kept


def _gradients(items):
    """The gradients among tensors, arrays and parameters, torch's own among them
    (those with one; one that is named twice, as a shared weight's may be, counts
    once), and the addresses of a list of tensors alone, else None."""
    items = list(items)
    if set(map(type, items)) == {torch.Tensor}:
        at = list(map(_data_ptr, items))
        return (items, at) if len(set(at)) == len(at) else (_distinct(items), None)
    found = [p if isinstance(p, (torch.Tensor, np.ndarray))
             and not isinstance(p, torch.nn.Parameter) else p.grad for p in items]
    return _distinct([g for g in found if g is not None]), None


def _uploaded(grads, at):
    """The gradients as contiguous tensors, arrays on the device, and their
    addresses."""
    def upload(g):
        if isinstance(g, np.ndarray):
            if g.dtype not in (np.float32, np.float64, np.float16):
                raise TypeError(f"gradients must be float arrays, got {g.dtype}")
            return torch.from_numpy(np.ascontiguousarray(g)).to(_device())
        return g.contiguous()

    if at is None or not all(map(_contiguous, grads)):
        grads = [upload(g) for g in grads]
        at = list(map(_data_ptr, grads))
    return grads, at


def grad_norm(gradients: Iterable) -> torch.Tensor:
    """The 2-norm over all elements of all gradients (device tensors, numpy
    arrays, or parameters, whose ``grad`` counts), a 0-d fp32 device tensor.
    Squares are summed in fp64; one gradient named twice counts once."""
    return _clip(*_uploaded(*_gradients(gradients)), None, 0.0, 0.0)


def clip_grad_norm(gradients: Iterable, max_norm: float, *, eps: float = 1e-6,
                   out: Optional[List[torch.Tensor]] = None) -> torch.Tensor:
    """Scales gradients by min(1, max_norm / (norm + eps)), norm being their
    common 2-norm, and returns that norm (a 0-d fp32 device tensor; nothing waits
    for the device unless a gradient is a numpy array).

    gradients: device tensors (fp32, f16, bf16, float64, mixed), numpy arrays, or
    parameters (torch.nn's too), whose ``grad`` is taken; those without one are passed over, and one
    named twice (a shared weight's) counts and is scaled once.  They are clipped in
    place, or, with ``out`` (for each that counts a contiguous device tensor of as
    many elements, of any of these types), written there: bf16 gradients to the
    fp32 ones an optimizer steps with in the same pass.  Contiguous ones that share
    memory otherwise, and outs that do, are a ValueError.  A NaN norm makes every
    gradient NaN.  Stands for the clipping of the reference's SGD
    (novann/optim/sgd.py:37-82), before any optimizer's step."""
    max_norm, eps = float(max_norm), float(eps)
    if not max_norm >= 0.0 or not eps >= 0.0:
        raise ValueError(f"max_norm and eps must not be negative, got {max_norm} and {eps}")
    found, at = _gradients(gradients)
    grads, at = _uploaded(found, at)
    if out is not None:
        outs = list(out)
        if len(outs) != len(grads):
            raise ValueError(f"{len(outs)} outputs for {len(grads)} gradients")
        if not all(map(_contiguous, outs)):
            raise ValueError("every out must be contiguous")
        return _clip(grads, at, outs, max_norm, eps)
    norm = _clip(grads, at, grads, max_norm, eps)
    if grads is found:
        return norm
    for g, d in zip(found, grads):
        if isinstance(g, np.ndarray):
            g[...] = d.cpu().numpy()
        elif d is not g:
            g.copy_(d)
    return norm
