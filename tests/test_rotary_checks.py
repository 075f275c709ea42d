"""What kmx_rotary_turns and kmx_rotary refuse before any device work, beside tests/test_around_cache.py."""
import ctypes

import numpy as np
import pytest

from test_around_cache import rows_of
from test_cache4 import DUMMY


@pytest.mark.parametrize("bad", [(128, 5e-324, 1.0, 0.0, 1.0, 32.0), (64, 1e4, 1e-310, 0.0, 1.0, 32.0), (64, 1e4, 1e-310, 16.0, 1.0, 32.0)])
def test_frequencies_beyond_a_double(km, bad):
    """A pair whose frequency is no finite number is refused, and nothing is written."""
    out = np.full(bad[0] // 2, 77, np.uint64)
    lib = km.hip_lib()
    assert lib.kmx_rotary_turns(*bad, out.ctypes.data) == km.KMX_ERR_INVALID_ARGUMENT and b"pair" in lib.kmx_last_error()
    assert np.all(out == 77)


def test_the_largest_frequencies_that_are_numbers(km):
    assert km.rotary_turns(64, 1e-300).shape == (32,) and km.rotary_turns(64, 1e4, 1e-300).shape == (32,)
    assert km.rotary_turns(256, 1e-310, 1.0, 4096.0, 1.0, 1e300).shape == (128,)  # (1e-310)^(-254 / 256) is 10^307.6, below the largest double


@pytest.mark.parametrize("which,off", [("turns", 4), ("turns", 1), ("positions", 2), ("positions", 1)])
def test_arrays_that_are_not_aligned(km, which, off):
    """On the device turns are numbers of 8 bytes and positions of 4."""
    at = dict(turns=DUMMY, positions=DUMMY)
    at[which] = ctypes.c_void_p((1 << 20) + off)
    lib = km.hip_lib()
    assert lib.kmx_rotary(km.TYPE_BF16, rows_of(km), 1, 5, 64, 32, at["turns"], at["positions"], 1, 0, 1.0) == km.KMX_ERR_INVALID_ARGUMENT and b"multiples" in lib.kmx_last_error()
