"""The C entries and the torch functions of the operators over feature rows, as far as no GPU is needed."""
import ctypes

import pytest

LL = ctypes.c_longlong


@pytest.fixture(scope="module")
def lib():
    from neuralgaussiansplatting_amd.diff_gaussian_rasterization import _lib
    L = _lib.lib()
    L.ngs_linear_slope_bytes.restype = ctypes.c_size_t
    L.ngs_last_error.restype = ctypes.c_char_p
    return L


def test_size_of_the_stored_derivative(lib):
    """Four bytes an element in every type, where the backward pass reads it; nothing where it forms z again."""
    f = lambda rows, k, n, dtype, act: lib.ngs_linear_slope_bytes(LL(rows), k, n, dtype, act)
    for dtype in range(3):
        assert f(300, 512, 512, dtype, 2) == 300 * 512 * 4
        assert f(1 << 22, 1024, 1024, dtype, 4) == 1 << 34
        assert f(300, 512, 512, dtype, 0) == 0 and f(300, 64, 64, dtype, 2) == 0
        assert f(0, 512, 512, dtype, 2) == 0 and f(-1, 512, 512, dtype, 2) == 0 and f(300, 512, 0, dtype, 2) == 0
    assert f(300, 512, 512, 3, 2) == 0
