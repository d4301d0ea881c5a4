"""Cast, amax and per-tensor quantization on device tensors.

Thin host layer over the C ABI: torch provides the device memory and the
current HIP stream, libnovaq.so does the work.  Element storage:

  f32 -> torch.float32, f16 -> torch.float16, bf16 -> torch.bfloat16,
  e4m3 -> torch.float8_e4m3fn, e5m2 -> torch.float8_e5m2,
  e2m1 -> torch.uint8 holding ceil(n/2) bytes (element 2i in the low nibble).

The rounding / special-value rules are the ones in include/novaq.h.
NovaNN itself has no cast API; its only conversion is ``astype(np.float32)``
at layer entry (novann/layers/linear/linear.py:81).
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import DTYPES, check

STORAGE = {
    "f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16,
    "e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2, "e2m1": torch.uint8,
}
QUANTIZED = ("e4m3", "e5m2", "e2m1")


def _dtype_code(name: str) -> int:
    try:
        return DTYPES[name]
    except KeyError:
        raise TypeError(f"unknown dtype '{name}', expected one of {tuple(DTYPES)}") from None


def storage_numel(dtype: str, n: int) -> int:
    """Number of storage elements holding n logical elements."""
    return (n + 1) // 2 if dtype == "e2m1" else n


_BITS = {"f32": 32, "f16": 16, "bf16": 16, "e4m3": 8, "e5m2": 8, "e2m1": 4}


def _require_holds(t: torch.Tensor, dtype: str, n: int, what: str) -> None:
    """ValueError unless t's storage holds n logical elements of dtype (the
    kernels would otherwise read or write past the end of the buffer)."""
    need = (n * _BITS[dtype] + 7) // 8
    have = t.numel() * t.element_size()
    if have < need:
        raise ValueError(f"{what} holds {have} bytes, {n} {dtype} elements need {need}")


def _stream(t: torch.Tensor) -> int:
    # (the address alone: building a torch Stream costs 1.9 us a call, this 0.1)
    return torch._C._cuda_getCurrentRawStream(t.get_device())


def _require_device(t: torch.Tensor, what: str) -> None:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{what} must be a CUDA (HIP) device tensor")
    if not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous")


def _aligned16(t: torch.Tensor) -> torch.Tensor:
    """t itself when its data starts on a 16-byte boundary (what the kernels'
    vector accesses need), else an aligned copy: a view into a larger tensor
    works, at the cost of the copy."""
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def dtype_of(t: torch.Tensor) -> str:
    for k, v in STORAGE.items():
        if t.dtype == v:
            return k
    raise TypeError(f"no novaq dtype is stored as {t.dtype}")


def cast(src: torch.Tensor, dst_dtype: str, *, src_dtype: Optional[str] = None,
         n: Optional[int] = None, scale: Optional[torch.Tensor] = None,
         out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Cast the n elements of ``src`` to ``dst_dtype``; returns a flat tensor.

    ``scale`` is a one-element fp32 device tensor s: quantizing encodes x/s
    (as x * (1/s)), dequantizing decodes q * s.  ``n`` defaults to the number
    of logical elements of src (2 per byte for e2m1)."""
    _require_device(src, "src")
    src_dtype = src_dtype or dtype_of(src)
    st, dt = _dtype_code(src_dtype), _dtype_code(dst_dtype)
    if n is None:
        n = src.numel() * 2 if src_dtype == "e2m1" else src.numel()
    n = int(n)
    if n < 0:
        raise ValueError(f"cast: negative element count {n}")
    _require_holds(src, src_dtype, n, "src")
    src = _aligned16(src)
    target = None
    if out is None:
        out = torch.empty(storage_numel(dst_dtype, n), dtype=STORAGE[dst_dtype],
                          device=src.device)
    else:
        _require_device(out, "out")
        if out.dtype != STORAGE[dst_dtype]:
            raise TypeError(f"out must be {STORAGE[dst_dtype]} for {dst_dtype}, got {out.dtype}")
        _require_holds(out, dst_dtype, n, "out")
        if out.data_ptr() % 16:
            # write into an aligned buffer, then copy into the caller's view
            target, out = out, torch.empty(storage_numel(dst_dtype, n),
                                           dtype=STORAGE[dst_dtype], device=src.device)
    if scale is not None:
        _require_device(scale, "scale")
        if scale.dtype != torch.float32:
            raise TypeError("scale must be float32")
    lib = _lib.load()
    check(lib.novaq_cast(src.data_ptr(), st, out.data_ptr(), dt, n, _ptr(scale),
                         _stream(src)), f"cast {src_dtype}->{dst_dtype}")
    if target is not None:
        target.reshape(-1)[:out.numel()].copy_(out)
        return target
    return out


def amax(x: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """NaN-ignoring max |x| as a one-element fp32 device tensor."""
    _require_device(x, "x")
    x = _aligned16(x)
    if out is None:
        out = torch.empty(1, dtype=torch.float32, device=x.device)
    check(_lib.load().novaq_amax(x.data_ptr(), _dtype_code(dtype_of(x)), x.numel(),
                                 out.data_ptr(), _stream(x)), "amax")
    return out


def scale_from_amax(a: torch.Tensor, dst_dtype: str) -> torch.Tensor:
    """s = amax / fmt_max (448 / 57344 / 6), or 1 if amax is 0 or not finite."""
    _require_device(a, "amax")
    out = torch.empty(1, dtype=torch.float32, device=a.device)
    check(_lib.load().novaq_scale_from_amax(a.data_ptr(), _dtype_code(dst_dtype),
                                            out.data_ptr(), _stream(a)), "scale_from_amax")
    return out


@dataclass
class Quantized:
    """Per-tensor quantized data: codes (flat storage), logical shape, dtype
    name and the device tensors amax and scale (one fp32 each)."""
    data: torch.Tensor
    shape: tuple
    dtype: str
    scale: torch.Tensor
    amax: Optional[torch.Tensor] = None

    @property
    def numel(self) -> int:
        n = 1
        for d in self.shape:
            n *= int(d)
        return n

    def check(self, what: str = "quantized tensor") -> None:
        """ValueError unless ``data`` holds the codes of prod(shape) elements."""
        if self.dtype not in QUANTIZED:
            raise TypeError(f"{what}: dtype must be one of {QUANTIZED}, got {self.dtype}")
        _require_device(self.data, f"{what} data")
        _require_holds(self.data, self.dtype, self.numel, f"{what} data")


def quantize(x: torch.Tensor, dst_dtype: str) -> Quantized:
    """amax -> s = amax / fmt_max -> encode(x * (1/s)), all on the device."""
    _require_device(x, "x")
    if dst_dtype not in QUANTIZED:
        raise TypeError(f"quantize target must be one of {QUANTIZED}")
    x = _aligned16(x)
    n = x.numel()
    data = torch.empty(storage_numel(dst_dtype, n), dtype=STORAGE[dst_dtype], device=x.device)
    st = torch.empty(2, dtype=torch.float32, device=x.device)
    check(_lib.load().novaq_quantize(x.data_ptr(), _dtype_code(dtype_of(x)), data.data_ptr(),
                                     _dtype_code(dst_dtype), n, st.data_ptr(), _stream(x)),
          f"quantize ->{dst_dtype}")
    return Quantized(data=data, shape=tuple(x.shape), dtype=dst_dtype, scale=st[1:2],
                     amax=st[0:1])


def dequantize(q: Quantized, dst_dtype: str = "f32") -> torch.Tensor:
    """decode(q) * s in the requested float type, reshaped to q.shape."""
    q.check()
    y = cast(q.data, dst_dtype, src_dtype=q.dtype, n=q.numel, scale=q.scale)
    return y.view(q.shape)


def pack_fp4(x: torch.Tensor, scale: Optional[torch.Tensor] = None) -> torch.Tensor:
    """fp32 -> E2M1, two elements per byte (element 2i in bits 3..0)."""
    if x.dtype != torch.float32:
        raise TypeError("pack_fp4 takes float32")
    return cast(x, "e2m1", scale=scale)


def unpack_fp4(packed: torch.Tensor, n: int, scale: Optional[torch.Tensor] = None
               ) -> torch.Tensor:
    """E2M1 bytes -> n fp32 values (times scale when given)."""
    return cast(packed, "f32", src_dtype="e2m1", n=n, scale=scale)


# --------------------------------------------------------------------------
# FP8 with a power-of-two scale for each block of 128

BLOCK = 128
BLOCK_DTYPES = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
_FLOATS = {torch.float32: DTYPES["f32"], torch.float16: DTYPES["f16"],
           torch.bfloat16: DTYPES["bf16"]}


def block_pitch(n: int) -> int:
    """Codes in a row of n elements: whole blocks."""
    return -(-n // BLOCK) * BLOCK


def block_groups(n: int) -> int:
    """Exponents in a row of n elements: one for 128, in whole fours."""
    return -(-n // (4 * BLOCK)) * 4


@dataclass
class BlockQuantized:
    """A matrix (rows, columns) as FP8 codes with a power-of-two scale for each block.

    data: codes (rows, columns rounded up to 128), zeros past the columns; exponents:
    uint8, one e for each 128 columns of a row (block_rows 1) or for 128 x 128 elements
    (block_rows 128), in rows of whole fours, the scale being 2^(e - 127).  transposed:
    the matrix is the transpose of the one it was made from (what a layer's backward
    keeps of its input).  lead: the shape that the rows have in a tensor of other than two
    dimensions (layer_norm's output), which a product's output has again; None: (rows,)."""
    data: torch.Tensor
    exponents: torch.Tensor
    shape: tuple
    dtype: str
    block_rows: int = 1
    transposed: bool = False
    lead: Optional[tuple] = None

    def check(self, what: str = "blocks") -> int:
        """ValueError or TypeError unless the tensors hold that matrix; their device's index."""
        if self.lead is not None and math.prod(self.lead) != self.shape[0]:
            raise ValueError(f"{what}: rows {tuple(self.lead)} are not the matrix's {self.shape[0]}")
        return check_blocks(self.data, self.exponents, self.shape, self.dtype, self.block_rows,
                            what)


def check_blocks(codes, exponents, shape, dtype, block_rows, what) -> int:
    """The index of the device that they are on."""
    rows, cols = shape
    at = codes.get_device()
    if codes.dtype is BLOCK_DTYPES.get(dtype) and exponents.dtype is torch.uint8 and \
            block_rows in (1, BLOCK) and at >= 0 and exponents.get_device() == at and \
            codes.shape == (rows, -(-cols // BLOCK) * BLOCK) and codes.is_contiguous() and \
            exponents.shape == (rows if block_rows == 1 else -(-rows // BLOCK),
                                -(-cols // (4 * BLOCK)) * 4) and exponents.is_contiguous():
        return at
    if codes.dtype is not BLOCK_DTYPES.get(dtype):
        raise TypeError(f"{what}: codes must be {' or '.join(BLOCK_DTYPES)}, got {dtype} in "
                        f"{codes.dtype}")
    if exponents.dtype is not torch.uint8:
        raise TypeError(f"{what}: exponents must be uint8, got {exponents.dtype}")
    if block_rows not in (1, BLOCK):
        raise ValueError(f"{what}: block_rows must be 1 or {BLOCK}, got {block_rows}")
    if at < 0 or exponents.get_device() != at:
        raise ValueError(f"{what}: codes and exponents must be on one CUDA (HIP) device")
    erows = rows if block_rows == 1 else -(-rows // BLOCK)
    raise ValueError(f"{what}: a {(rows, cols)} matrix has contiguous codes "
                     f"{(rows, block_pitch(cols))} and exponents {(erows, block_groups(cols))}, "
                     f"got {tuple(codes.shape)} and {tuple(exponents.shape)}")


_raw_stream, _current_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice


def on_device(dev, fn, *args) -> int:
    """fn(*args, stream) with the device (or its index) current, on its current stream."""
    at = dev if type(dev) is int else dev.index
    stream = _raw_stream(at)
    if _current_device() == at:
        return fn(*args, stream)
    with torch.cuda.device(at):
        return fn(*args, stream)


def _matrix(x: torch.Tensor, what: str) -> torch.Tensor:
    """A 2-D float device tensor as the kernels read it."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise ValueError(f"{what} must be a CUDA (HIP) device tensor")
    if x.dtype not in _FLOATS:
        raise TypeError(f"{what} must be fp32, f16 or bf16, got {x.dtype}")
    if x.dim() != 2:
        raise ValueError(f"{what} must be 2-D, got shape {tuple(x.shape)}")
    return _aligned16(x.contiguous())


def make_blocks(x: torch.Tensor, dtype: str, block_rows: int = 1, *, rows: bool = True,
                transposed: bool = False, colsum: bool = False
                ) -> Tuple[Optional[BlockQuantized], Optional[BlockQuantized],
                           Optional[torch.Tensor]]:
    """(x in blocks, its transpose in blocks, the sums of its columns), each where asked
    for, from one read of x (a matrix as ``_matrix`` gives it)."""
    if dtype not in BLOCK_DTYPES:
        raise TypeError(f"blocks are {' or '.join(BLOCK_DTYPES)}, got {dtype!r}")
    R, C = x.shape
    dev, f8 = x.device, BLOCK_DTYPES[dtype]

    def empty(r, c):
        er = r if block_rows == 1 else -(-r // BLOCK)
        return BlockQuantized(torch.empty((r, block_pitch(c)), dtype=f8, device=dev),
                              torch.empty((er, block_groups(c)), dtype=torch.uint8, device=dev),
                              (r, c), dtype, block_rows)

    q = empty(R, C) if rows else None
    t = empty(C, R) if transposed else None
    if t is not None:
        t.transposed = True
    sums = torch.empty(C, dtype=torch.float32, device=dev) if colsum else None
    lib = _lib.load()
    nbytes = lib.novaq_quantize_blocks_workspace(R, C) if colsum else 0
    work = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    check(on_device(dev, lib.novaq_quantize_blocks, x.data_ptr(), _FLOATS[x.dtype], R, C,
                    DTYPES[dtype], block_rows, None if q is None else q.data.data_ptr(),
                    None if q is None else q.exponents.data_ptr(),
                    None if t is None else t.data.data_ptr(),
                    None if t is None else t.exponents.data_ptr(), _ptr(sums), _ptr(work),
                    nbytes), "quantize blocks")
    return q, t, sums


def quantize_blocks(x: torch.Tensor, dst_dtype: str = "e4m3", block_rows: int = 1
                    ) -> BlockQuantized:
    """A float matrix as FP8 codes with a power-of-two scale for each 128 columns of a
    row, or (block_rows 128) for 128 x 128 elements: the smallest scale with the block's
    largest magnitude within the format's, 1 for zeros (and for a block with an infinity,
    which saturates)."""
    if block_rows not in (1, BLOCK):
        raise ValueError(f"block_rows must be 1 or {BLOCK}, got {block_rows}")
    return make_blocks(_matrix(x, "x"), dst_dtype, block_rows)[0]


def dequantize_blocks(q: BlockQuantized, dst_dtype: str = "f32") -> torch.Tensor:
    """code * 2^(e - 127) in 'f32', 'bf16' or 'f16', of the matrix's shape."""
    q.check()
    if dst_dtype not in ("f32", "bf16", "f16"):
        raise TypeError(f"blocks decode to f32, bf16 or f16, got {dst_dtype!r}")
    out = torch.empty(q.shape, dtype=STORAGE[dst_dtype], device=q.data.device)
    check(on_device(out.device, _lib.load().novaq_dequantize_blocks, q.data.data_ptr(),
                    DTYPES[q.dtype], q.exponents.data_ptr(), q.shape[0], q.shape[1],
                    q.block_rows, out.data_ptr(), DTYPES[dst_dtype]), "dequantize blocks")
    return out
