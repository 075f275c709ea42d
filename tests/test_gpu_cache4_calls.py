"""Calls around the kernels of the 4-bit cache: bounds that say little, work space, recordings (-m gpu)."""
import numpy as np
import pytest

from test_gpu_cache4 import BF16, Cache, Queries, bound_all, choice, device, select

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("group", [2, 20])
@pytest.mark.parametrize("counts", [[1, 1], [40, 3]])
def test_bounds_on_queries_that_say_nothing(km, gpu, group, counts):
    """max_queries may be any number from the largest count on."""
    rng = np.random.default_rng(group)
    c = Cache(km, rng, 2, 64, 16, 70)
    s = Queries(km, rng, c, [900, 120], counts, group, BF16).fill(rng)
    want = bound_all(s)
    for most in (70000, 1 << 24, (1 << 32) - 1):
        s.batch = km.Cache4Batch(2, 2 * group, s.tokens, most, 900, device(km, s.starts), device(km, np.int32(s.lengths)), device(km, s.table), s.table.shape[1])
        s.c.dev.reserve(s.batch, 6)
        s.check()
        chosen = select(s, 6, 1, 1)
        assert np.array_equal(chosen, choice(s, want, 6, 1, 1, True))
        s.check(chosen=chosen)
