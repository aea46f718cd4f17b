"""The workspace of a layer norm's gradient over every column count."""

import ctypes as C

import pytest

from quabla_b200 import _lib

# 296 partial rows of weight and bias gradients in float32 at 4096 columns (float64: 148 at 4096).
LARGEST = 9_699_328


@pytest.mark.parametrize("dtype,most,item", [(_lib.F32, 65536, 4), (_lib.F64, 32768, 8), (_lib.F16, 65536, 4), (_lib.BF16, 65536, 4)])
def test_workspace_of_every_column_count(dtype, most, item):
    lib, size, seen = _lib.load(), C.c_size_t(), 0
    at = C.byref(size)
    for cols in range(1, most + 1):
        assert lib.qb200_layer_norm_workspace(dtype, 1 << 40, cols, at) == _lib.OK
        # Whole partial rows, at most two for each multiprocessor.
        assert size.value % (2 * cols * item) == 0 and 1 <= size.value // (2 * cols * item) <= 296
        seen = max(seen, size.value)
    assert seen == LARGEST


@pytest.mark.parametrize("dtype,most", [(_lib.F32, 65536), (_lib.F64, 32768), (_lib.BF16, 65536)])
def test_workspace_grows_with_the_rows_up_to_its_bound(dtype, most):
    lib, size = _lib.load(), C.c_size_t()
    for cols in (1, 15, 16, 17, 500, 4096, 4097, 8193, most):
        last = 0
        for rows in [0, 1, 2, 3, 7, 100, 1000, 10**4, 10**5, 10**6, 1 << 40]:
            _lib.check(lib.qb200_layer_norm_workspace(dtype, rows, cols, C.byref(size)))
            assert last <= size.value <= LARGEST and (size.value > 0) == (rows > 0)
            last = size.value
