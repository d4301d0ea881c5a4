"""AdamW with NovaNN's interface (novann/optim/adamw.py:6-69), on the GPU.

Same constructor (parameters, lr, betas, weight_decay, epsilon), ``step`` and
``zero_grad``; BatchNorm gamma / beta (by name) are not decayed, as there.
Each step is the float32 update the reference computes on its float32 arrays,
bit for bit (libnovaq ``novaq_adamw_step``).  ``QuantizedParameters`` step
their fp32 ``master`` weights and re-quantize their codes and scale in the
same call (``novaq_adamw_requantize``).  ``Parameters`` holding numpy arrays
are uploaded at every step (so changes a caller makes to ``.data`` between
steps count, as with the reference), stepped on the device and written back
in place.  float64 arrays (the BatchNorm gamma / beta, float64 in the
reference too) keep float64 moments and step in float64 with numpy's
promotion of a float32 gradient (``novaq_adamw_step_f64``); any other numpy
array steps in float32 (the reference's float32 parameters).
"""
from __future__ import annotations

import ctypes
import math
from array import array
from operator import attrgetter
from typing import Iterable, List, Optional

import numpy as np
import torch

from . import _lib
from ._lib import DTYPES, check
from .module import Parameters, QuantizedParameters


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


class AdamW:
    """AdamW with decoupled weight decay (adamw.py:6-69)."""

    def __init__(self, parameters: Iterable, lr: float, betas=(0.9, 0.999),
                 weight_decay: float = 0, epsilon: float = 1e-8) -> None:
        self.params: List = list(parameters)
        self.lr, self.wd = float(lr), float(weight_decay)
        self.b1, self.b2 = float(betas[0]), float(betas[1])
        self.eps = float(epsilon)
        self.t = 0
        dev = _device()
        self._w: List[torch.Tensor] = []
        for p in self.params:
            if isinstance(p, QuantizedParameters):
                if p.master is None:
                    raise ValueError("AdamW: a QuantizedParameters needs fp32 master weights "
                                     "(QuantizedParameters.from_float(..., keep_master=True))")
                self._w.append(p.master)
            elif _is_f64(p):
                self._w.append(torch.from_numpy(np.ascontiguousarray(p.data)).to(dev))
            elif isinstance(p.data, np.ndarray):
                self._w.append(_dev_f32(p.data, dev))
            else:
                if p.data.dtype != torch.float32 or not p.data.is_contiguous():
                    raise TypeError("AdamW: device parameters must be contiguous float32")
                self._w.append(p.data)
        self.m_t = [torch.zeros_like(w) for w in self._w]
        self.v_t = [torch.zeros_like(w) for w in self._w]
        self._amax_scale: List[Optional[torch.Tensor]] = [
            torch.empty(2, dtype=torch.float32, device=dev)
            if isinstance(p, QuantizedParameters) else None for p in self.params]

    def step(self) -> None:
        """One optimization step (adamw.py:41-65)."""
        self.t += 1
        lib = _lib.load()
        for i, p in enumerate(self.params):
            if p.grad is None:
                continue
            w = self._w[i]
            if isinstance(getattr(p, "data", None), np.ndarray):
                # the caller may have changed .data since the last step
                w.copy_(torch.from_numpy(np.ascontiguousarray(p.data).reshape(w.shape).astype(
                    np.float64 if w.dtype == torch.float64 else np.float32, copy=False)))
            is_bn_param = getattr(p, "name", None) in ("gamma", "beta")
            hp = _lib.AdamW(self.lr, self.b1, self.b2, self.eps, self.wd, self.t,
                            0 if is_bn_param else 1)
            # (the raw lookup below takes a host tensor's device as "the current
            # one"; the kernels would then follow host pointers)
            if not w.is_cuda:
                raise ValueError(f"AdamW: parameters must be CUDA (HIP) device tensors, got one "
                                 f"on {w.device}")
            stream = torch._C._cuda_getCurrentRawStream(w.get_device())
            if w.dtype == torch.float64:
                g, g32 = _dev_grad64(p.grad, w.device)
                if g.numel() != w.numel():
                    raise ValueError(f"AdamW: gradient of {g.numel()} values for a parameter "
                                     f"of {w.numel()}")
                check(lib.novaq_adamw_step_f64(
                    w.data_ptr(), g.data_ptr(), int(g32), self.m_t[i].data_ptr(),
                    self.v_t[i].data_ptr(), w.numel(), ctypes.byref(hp), stream), "adamw f64")
                p.data[...] = w.cpu().numpy().reshape(p.data.shape)
                continue
            g = _dev_f32(p.grad, w.device)
            if isinstance(p, QuantizedParameters) and p.stored_shape != p.shape:
                # the pad column of an odd-width E2M1 weight: zero gradient
                g = torch.nn.functional.pad(g.reshape(p.shape), (0, 1))
            g = g.reshape(w.shape)
            if isinstance(p, QuantizedParameters):
                st = self._amax_scale[i]
                check(lib.novaq_adamw_requantize(
                    w.data_ptr(), g.data_ptr(), self.m_t[i].data_ptr(), self.v_t[i].data_ptr(),
                    w.numel(), ctypes.byref(hp), p.codes.data_ptr(), DTYPES[p.dtype],
                    st.data_ptr(), stream), "adamw requantize")
                # the codes and scale the products read now follow the master
                # (the next step rewrites st after this step's readers, in
                # stream order)
                p.amax, p.scale = st[0:1], st[1:2]
            else:
                check(lib.novaq_adamw_step(
                    w.data_ptr(), g.data_ptr(), self.m_t[i].data_ptr(), self.v_t[i].data_ptr(),
                    w.numel(), ctypes.byref(hp), None, stream), "adamw step")
                if isinstance(p.data, np.ndarray):
                    p.data[...] = w.cpu().numpy().reshape(p.data.shape)

    def zero_grad(self, set_to_none: bool = False) -> None:
        """Clears the gradients of all optimized parameters (adamw.py:67-70)."""
        for p in self.params:
            p.zero_grad(set_to_none=set_to_none)


_GRAD_TYPES = {torch.float32: DTYPES["f32"], torch.float16: DTYPES["f16"],
               torch.bfloat16: DTYPES["bf16"], torch.float64: _lib.F64}


# (what follows handles hundreds of tensors a call: whole lists at a time, a
# few tenths of a microsecond a tensor)
_data_ptr, _numel = torch.Tensor.data_ptr, torch.Tensor.numel
_contiguous = torch.Tensor.is_contiguous
_dtype, _is_cuda = attrgetter("dtype"), attrgetter("is_cuda")


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
