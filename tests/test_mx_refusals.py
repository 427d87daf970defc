"""What the MX product refuses on the host, by its C entry point."""

import ctypes

import pytest

from tests.test_library import LIBRARY
from tests.test_mx import needs_library


@needs_library
@pytest.mark.parametrize("op,length", [(1, 4), (2, 8), (4, 4), (5, 8)])
@pytest.mark.parametrize("kind,size", [(0, 4), (16, 2), (32, 2)])
def test_the_product_refuses_a_result_over_its_epilogues_vectors(op, length, kind, size):
    """A tile's store would change what later tiles read: row vectors have M elements, column vectors N."""
    library = ctypes.CDLL(str(LIBRARY))
    library.krn_amd_last_error.restype = ctypes.c_char_p
    p, i64 = ctypes.c_void_p, ctypes.c_int64
    c, m, n = 1 << 40, 4, 8
    for vector in (c, c + m * n * 2 - 2, c - length * size + 2):
        assert library.krn_mx_gemm(p(1 << 30), p(1 << 32), p(1 << 33), p(1 << 34), p(c), 2, i64(m), i64(n), i64(64), 1,
                                   (ctypes.c_int * 1)(op + kind), None, (p * 1)(vector), None, i64(0), None) == -1
        assert "shares memory" in library.krn_amd_last_error().decode()
