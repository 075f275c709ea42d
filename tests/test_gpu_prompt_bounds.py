"""Bounds of the attention over prompts that ask for more work-groups than a launch has (-m gpu)."""
import numpy as np
import pytest

from test_gpu_cache4 import BF16, device

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128, 192])
def test_too_many_sequences_of_too_many_queries(km, gpu, dim):
    """The call says so, and the library goes on: 2^20 queries a sequence by their bound, 512 of them, none of which has any."""
    sequences, queries = 512, 1 << 20
    starts = device(km, np.zeros(sequences + 1, np.int32))
    rows, out = device(km, np.zeros(4 * dim, np.uint16)), device(km, np.full(4 * dim, 0x5A5A, np.uint16))
    prompt = km.Prompt(sequences, 4, 1, dim, queries, 1, queries, 1, starts, starts)
    with pytest.raises(km.KmxError) as e:
        prompt.attend(BF16, rows, rows, rows, out, 1.0)
    assert e.value.code == km.KMX_ERR_UNSUPPORTED and "512 sequences of up to 1048576 queries" in str(e.value)
    one = km.Prompt(1, 4, 1, dim, 1, 1, 1, 1, *(device(km, np.int32([0, 1])) for _ in range(2)))
    one.attend(BF16, rows, rows, rows, out, 1.0)
    km.sync()
    assert not out.read(np.uint16, 4 * dim).any()
