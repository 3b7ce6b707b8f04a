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
