"""Attention to shared prefixes with more sequences than a launch has room for (-m gpu)."""
import numpy as np
import pytest

from test_gpu_cache4 import BF16, Cache, device

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("many", ["own", "prefixes"])
def test_too_many_sequences_behind_a_prefix(km, gpu, many):
    """Refused by its own name, before anything is launched: rows and sums stay as they were."""
    rng = np.random.default_rng(1)
    n = 70000
    c = Cache(km, rng, 1, 32, 16, 2)
    q, out, lse = device(km, np.zeros((n, 32), np.uint16)), device(km, np.full((n, 32), 0x5A5A, np.uint16)), device(km, np.full(n, 77, np.float32))
    table = device(km, np.zeros((n, 1), np.int32))
    alone = km.Cache4Batch(n, 1, n, 1, 16, device(km, np.arange(n + 1, dtype=np.int32)), device(km, np.full(n, 9, np.int32)), table, 1)
    whole = km.Cache4Batch(1, 1, n, n, 16, device(km, np.int32([0, n])), device(km, np.int32([9])), table, 1)
    with pytest.raises(km.KmxError) as e:
        c.dev.attend_shared(*((whole, alone) if many == "own" else (alone, whole)), BF16, q, out, 1.0, lse=lse)
    assert e.value.code == km.KMX_ERR_UNSUPPORTED and "kmx_cache4_attend_shared: 70000 sequences" in str(e.value)
    with pytest.raises(km.KmxError) as e:
        c.dev.attend(alone, BF16, q, out, 1.0, lse=lse)
    assert "kmx_cache4_attend: 70000 sequences" in str(e.value)
    km.sync()
    assert np.all(out.read(np.uint16, 32 * n) == 0x5A5A) and np.all(lse.read(np.float32, n) == 77)
