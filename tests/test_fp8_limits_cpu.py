"""The largest sizes that the 8-bit float entry points take: refusals, before any CUDA call."""
import ctypes

import pytest

from llima_b200 import _native as N

SIZE, P = -2, 0x1000   # P: a 16-byte-aligned address that no call here may read


@pytest.mark.parametrize("fmt,unit,size", [(8, 32, 34), (2, 32, 18), (12, 256, 144), (14, 256, 210), (0, 1, 4), (30, 1, 2)])
@pytest.mark.parametrize("cols", [1 << 31, 1 << 32, (1 << 32) + 256, 1 << 37])
def test_rows_of_more_columns_than_32_bits_hold(fmt, unit, size, cols):
    """A tile's place in its row is a 32-bit number."""
    t = N.Tensor(type=fmt, rows=1, cols=cols, src=P, src_bytes=cols // unit * size, codes=P)
    assert N.lib().gq_convert_fp8(ctypes.byref(t), P, None) == SIZE
