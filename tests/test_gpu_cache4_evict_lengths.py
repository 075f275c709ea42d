"""Eviction where a length on the device says nothing: weights and rows of the sequences beside it, too (-m gpu)."""
import numpy as np
import pytest

from test_gpu_cache4 import device
from test_gpu_cache4_evict import Evict

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("said", [[100, -7], [-1, 100], [100, -2 ** 31], [0, 0]])
def test_lengths_below_zero_are_none(km, gpu, said):
    rng = np.random.default_rng(3)
    e = Evict(km, rng, 2, 64, 16, [100, 100], 30, 2, 4)
    e.batch = km.Cache4Batch(2, 2, 0, 0, 100, device(km, e.s.starts), device(km, np.int32(said)), device(km, e.s.table), e.s.table.shape[1])
    e.lengths = [max(0, n) for n in said]
    got = e.check()
    assert got[1].tolist() == [min(30, n) for n in e.lengths]
