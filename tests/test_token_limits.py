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
