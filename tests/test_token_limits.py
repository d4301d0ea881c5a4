"""Sizes whose launches would have 2^32 threads or more are refused before HIP is
touched, with the status for what is not supported."""
import pytest

from novann_amd import _lib

FAKE = 0x10000  # never dereferenced: every call below fails validation first


@pytest.mark.parametrize("N,D,V", [((1 << 27) + 1, 8, 100), (10, 8, (1 << 31) - 255),
                                   (1 << 24, 1 << 13, 100), (10, 1 << 20, 1 << 21)])
def test_linear_cross_entropy(N, D, V):
    lib = _lib.load()
    assert lib.novaq_linear_cross_entropy(FAKE, 2, N, D, FAKE, 2, None, V, FAKE, 64, -100, 1,
                                          FAKE, FAKE, FAKE, 1 << 62, None) == _lib.ENOTSUP
    assert lib.novaq_linear_cross_entropy_backward(
        FAKE, 2, N, D, FAKE, 2, None, V, FAKE, 64, -100, 1, None, FAKE, FAKE, FAKE, 2, FAKE,
        1 << 62, None) == _lib.ENOTSUP
    assert lib.novaq_linear_cross_entropy_workspace(N, D, V, 2, 2) == 256
    assert lib.novaq_linear_cross_entropy_backward_workspace(N, D, V, 2, 2) == 256


@pytest.mark.parametrize("N,D,V", [(1 << 27, 8, 100), (10, 8, (1 << 31) - 256),
                                   (1 << 22, 8, 1 << 18)])
def test_the_largest_have_a_workspace(N, D, V):
    lib = _lib.load()
    assert lib.novaq_linear_cross_entropy_workspace(N, D, V, 2, 2) > 256
    assert lib.novaq_linear_cross_entropy_backward_workspace(N, D, V, 2, 2) > 256


def test_embedding_backward():
    lib = _lib.load()

    def call(N):
        return lib.novaq_embedding_backward(FAKE, 0, FAKE, 64, N, 50, 8, 1.0, 0, FAKE, 0, FAKE,
                                            1 << 62, None)

    assert call(1 << 30) == _lib.ENOTSUP
    assert call((1 << 31) - 1025) == _lib.ENOTSUP
    assert lib.novaq_embedding_backward_workspace(1 << 30, 50, 8) == 0
    assert lib.novaq_embedding_backward_workspace((1 << 30) - 1, 50, 8) > 1 << 32
