"""Sizes at the limits that the row operators' header states, refused before anything reaches a GPU."""
import ctypes

import ogl_amd  # noqa: F401
from ogl_amd import _lib


def test_products_of_more_columns_than_a_launch_takes():
    """Up to 16 rows: 512 threads for 16 columns, so 2^27 of them are 2^32 threads.  More rows: column indexes of whole tiles stay below 2^31."""
    h = _lib.lib()
    buf = (ctypes.c_char * 256)()
    p = (ctypes.addressof(buf) + 63) // 64 * 64
    for M, N in [(1, 2 ** 27), (16, 2 ** 31 - 1), (17, 2 ** 31 - 1), (100, 2 ** 31 - 100)]:
        assert h.ogl_linear_i8(p, 64, p, None, 200, M, 40, p, 64, p, N, None, 0, p, N, 0, None) == -1, (M, N)
