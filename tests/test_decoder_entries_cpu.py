"""The C entries and the torch functions of the operators over feature rows, as far as no GPU is needed."""
import ctypes
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
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


def test_assembly_names_the_registers_it_writes():
    """Every inline assembly of the library that writes m0 says so to the compiler, which may keep a value there."""
    csrc = os.path.join(ROOT, "neuralgaussiansplatting_amd", "csrc")
    found = 0
    for folder, _, names in os.walk(csrc):
        for name in names:
            if not name.endswith((".hip", ".h")):
                continue
            with open(os.path.join(folder, name)) as f:
                text = f.read()
            for statement in re.findall(r"\basm\b[^;]*;", text):
                if re.search(r"\bs_mov_b32 m0\b", statement):
                    found += 1
                    clobbers = statement.rsplit(":", 1)[1]
                    assert '"m0"' in clobbers, name + ": " + statement
    assert found > 0


def test_column_sums_that_one_launch_does_not_hold_are_refused(lib):
    """Widths whose gradient sums would take 2^32 threads are refused before anything is launched."""
    some, none = ctypes.c_void_p(4096), None  # (an address that is never used)

    def norm(rows, width, dw, db):
        return lib.ngs_layer_norm_backward(LL(rows), width, 0, 0, some, LL(width), none, some, some, some, LL(width), none, dw, db,
                                           some, none)

    def linear(rows, n, db):
        return lib.ngs_linear_backward(LL(rows), 8, n, 0, 0, some, LL(8), some, LL(8), none, none, some, LL(n), none, none, db, some,
                                       none)

    for call in (lambda: norm(4, 1 << 28, some, none), lambda: norm(4, 1 << 30, none, some), lambda: norm(0, 1 << 28, some, some),
                 lambda: linear(4, (1 << 28) + 1, some), lambda: linear(0, 1 << 30, some)):
        assert call() == 1
        assert b"too many elements for one launch" in lib.ngs_last_error()
