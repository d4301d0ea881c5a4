"""What the token operators' C entry points refuse before they touch HIP."""
import ctypes
from array import array

import pytest

from novann_amd import _lib

FAKE = 0x10000  # never dereferenced: every call below fails validation first


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


# (ids, bits, N, table, w_dtype, w_scale, V, D, factor, out, out_dtype, stream)
@pytest.mark.parametrize("args,status", [
    ((FAKE, 64, 4, FAKE, 9, None, 8, 8, 1.0, FAKE, 0, None), _lib.EDTYPE),
    ((FAKE, 64, 4, FAKE, 0, None, 8, 8, 1.0, FAKE, 3, None), _lib.EDTYPE),   # FP8 output
    ((FAKE, 16, 4, FAKE, 0, None, 8, 8, 1.0, FAKE, 0, None), _lib.EDTYPE),   # 16-bit ids
    ((FAKE, 64, 4, FAKE, 0, FAKE, 8, 8, 1.0, FAKE, 0, None), _lib.EINVAL),   # scale on fp32
    ((FAKE, 64, -1, FAKE, 0, None, 8, 8, 1.0, FAKE, 0, None), _lib.EINVAL),
    ((FAKE, 64, 4, FAKE, 0, None, -8, 8, 1.0, FAKE, 0, None), _lib.EINVAL),
    ((FAKE, 64, 4, FAKE, 0, None, 0, 8, 1.0, FAKE, 0, None), _lib.ESHAPE),
    ((FAKE, 64, 4, FAKE, 0, None, 8, 0, 1.0, FAKE, 0, None), _lib.ESHAPE),
    ((FAKE, 64, 4, FAKE, 0, None, 1 << 31, 8, 1.0, FAKE, 0, None), _lib.ENOTSUP),
    ((FAKE + 4, 64, 4, FAKE, 0, None, 8, 8, 1.0, FAKE, 0, None), _lib.EALIGN),
    ((FAKE, 64, 4, FAKE + 8, 0, None, 8, 8, 1.0, FAKE, 0, None), _lib.EALIGN),
    ((FAKE, 64, 4, FAKE, 0, None, 8, 8, 1.0, FAKE + 8, 0, None), _lib.EALIGN),
    ((FAKE, 64, 4, None, 0, None, 8, 8, 1.0, FAKE, 0, None), _lib.EINVAL),
    ((FAKE, 64, 4, FAKE, 0, None, 8, 8, 1.0, None, 0, None), _lib.EINVAL),
    ((None, 64, 0, None, 0, None, 8, 8, 1.0, None, 0, None), _lib.OK),       # no tokens
])
def test_embedding(lib, args, status):
    assert lib.novaq_embedding(*args) == status


def test_embedding_backward(lib):
    ws = lib.novaq_embedding_backward_workspace(100, 50, 16)
    assert ws > 0
    assert lib.novaq_embedding_backward_workspace(0, 50, 16) == 0
    assert lib.novaq_embedding_backward_workspace(100, 0, 16) == 0

    def call(grad=FAKE, gdt=0, ids=FAKE, bits=64, N=100, V=50, D=16, out=FAKE, odt=0, work=FAKE,
             size=ws):
        return lib.novaq_embedding_backward(grad, gdt, ids, bits, N, V, D, 1.0, 0, out, odt, work,
                                            size, None)

    assert call(gdt=3) == _lib.EDTYPE
    assert call(odt=5) == _lib.EDTYPE
    assert call(bits=8) == _lib.EDTYPE
    assert call(N=-1) == _lib.EINVAL
    assert call(V=0) == _lib.ESHAPE
    assert call(N=(1 << 31) - 1) == _lib.ENOTSUP
    assert call(out=None) == _lib.EINVAL
    assert call(grad=None) == _lib.EINVAL
    assert call(grad=FAKE + 2) == _lib.EALIGN
    assert call(ids=FAKE + 4) == _lib.EALIGN
    assert call(work=FAKE + 8) == _lib.EALIGN
    assert call(work=None) == _lib.EINVAL
    assert call(size=ws - 1) == _lib.EINVAL


def test_linear_cross_entropy(lib):
    ws = lib.novaq_linear_cross_entropy_workspace(10, 64, 100, 2, 3)
    bws = lib.novaq_linear_cross_entropy_backward_workspace(10, 64, 100, 2, 3)
    assert ws > 0 and bws > 0

    def fwd(x=FAKE, xdt=2, N=10, D=64, w=FAKE, wdt=3, ws_=None, V=100, t=FAKE, bits=64, red=1,
            loss=FAKE, lse=FAKE, work=FAKE, size=ws):
        return lib.novaq_linear_cross_entropy(x, xdt, N, D, w, wdt, ws_, V, t, bits, -100, red,
                                              loss, lse, work, size, None)

    assert fwd(xdt=3) == _lib.EDTYPE                  # FP8 activations
    assert fwd(wdt=6) == _lib.EDTYPE
    assert fwd(bits=33) == _lib.EDTYPE
    assert fwd(wdt=0, ws_=FAKE) == _lib.EINVAL        # a scale on fp32
    assert fwd(red=3) == _lib.EINVAL
    assert fwd(N=-1) == _lib.EINVAL
    assert fwd(D=0) == _lib.ESHAPE
    assert fwd(V=0) == _lib.ESHAPE
    assert fwd(D=(1 << 20) + 1) == _lib.ENOTSUP
    assert fwd(x=None) == _lib.EINVAL
    assert fwd(w=None) == _lib.EINVAL
    assert fwd(t=None) == _lib.EINVAL
    assert fwd(t=FAKE + 4) == _lib.EALIGN
    assert fwd(x=FAKE + 8) == _lib.EALIGN
    assert fwd(loss=None) == _lib.EINVAL
    assert fwd(lse=None) == _lib.EINVAL
    assert fwd(work=None) == _lib.EINVAL
    assert fwd(work=FAKE + 8) == _lib.EALIGN
    assert fwd(size=ws - 1) == _lib.EINVAL
    assert fwd(N=0, x=None, t=None, loss=None, red=0) == _lib.OK

    def bwd(gw=FAKE, gx=FAKE, gdt=2, lse=FAKE, work=FAKE, size=bws, N=10):
        return lib.novaq_linear_cross_entropy_backward(
            FAKE, 2, N, 64, FAKE, 3, None, 100, FAKE, 64, -100, 1, None, lse, gx, gw, gdt, work,
            size, None)

    assert bwd(gdt=4) == _lib.EDTYPE
    assert bwd(gx=FAKE + 8) == _lib.EALIGN
    assert bwd(gw=FAKE + 8) == _lib.EALIGN
    assert bwd(lse=None) == _lib.EINVAL
    assert bwd(work=None) == _lib.EINVAL
    assert bwd(size=bws - 1) == _lib.EINVAL
    assert bwd(gx=None, gw=None, work=None, size=0) == _lib.OK   # nothing asked for
    assert bwd(N=0, gw=None) == _lib.OK


def test_clip_grad_norm(lib):
    ws = lib.novaq_clip_grad_norm_workspace(1)
    assert ws > 0 and lib.novaq_clip_grad_norm_workspace(1000) > ws

    def call(grad=FAKE, out=FAKE, n=10, gdt=0, odt=0, count=1, top=1.0, eps=0.0, norm=FAKE,
             work=FAKE, size=ws, rows=True):
        table = array("q", [grad, out, n, gdt | odt << 32])
        return lib.novaq_clip_grad_norm(table.buffer_info()[0] if rows else None, count, top, eps,
                                        norm, work, size, None)

    assert call(gdt=3) == _lib.EDTYPE
    assert call(odt=5) == _lib.EDTYPE
    assert call(n=-1) == _lib.EINVAL
    assert call(grad=0) == _lib.EINVAL
    assert call(count=-1) == _lib.EINVAL
    assert call(rows=False) == _lib.EINVAL
    assert call(top=-1.0) == _lib.EINVAL
    assert call(top=float("nan")) == _lib.EINVAL
    assert call(eps=-1.0) == _lib.EINVAL
    assert call(norm=None) == _lib.EINVAL
    assert call(work=None) == _lib.EINVAL
    assert call(size=ws - 1) == _lib.EINVAL
    assert call(grad=FAKE + 2) == _lib.EALIGN
    assert call(grad=FAKE + 4, gdt=6) == _lib.EALIGN
    assert call(out=FAKE + 1, odt=2) == _lib.EALIGN
    assert call(work=FAKE + 8) == _lib.EALIGN
    assert ctypes.sizeof(ctypes.c_void_p) == 8  # the rows above are the struct's layout
