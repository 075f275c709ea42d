"""Attention over prompts by eight wavefronts of 32 rows, which heads of 96 and 128 channels take where there are many rows (csrc/prompt_plan.h), against its definition in 64 bits (-m gpu).
That these batches are taken so is held by tests/test_prompt_plan.py."""
import numpy as np
import pytest

from test_gpu_cache4 import BF16, F16
from test_gpu_prompt import Prompts
from test_gpu_prompt_masks import Masked

pytestmark = pytest.mark.gpu

HEADS, GROUP = 2, 8
COUNTS = [300, 1, 2, 40, 7, 0, 65, 33, 64, 9, 3, 100, 5, 17, 31, 128]                # queries of a sequence
LENGTHS = [300, 1, 200, 40, 300, 9, 65, 70, 64, 0, 1, 333, 5, 17, 31, 128]          # and tokens: some longer, one without, one with fewer
DIMS = [96, 128]


def batch(km, rng, dim, kind, made=Prompts, **other):
    return made(km, rng, HEADS, GROUP, dim, COUNTS, LENGTHS, kind, extra=(1, 2), most=(1 << 20, 0), **other)  # (the bound on queries is all of them)


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dim", DIMS)
def test_many_rows(km, gpu, kind, causal, dim):
    rng = np.random.default_rng(dim)
    s = batch(km, rng, dim, kind)
    first = s.check(causal)
    for how in (dict(gaps=(8, 32), key_gaps=(0, 8), out_gaps=(16, 8), offset=8), dict(gaps=(1, 2), key_gaps=(3, 0), out_gaps=(3, 1), offset=1)):
        again = s.check(causal, **how)
        assert np.array_equal(first[0], again[0]) and np.array_equal(first[1], again[1])


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("loud", [1.0, 8.0])
def test_rising_and_masked_scores(km, gpu, kind, dim, loud):
    rng = np.random.default_rng(dim + 1)
    s = batch(km, rng, dim, kind, Masked, hidden=np.concatenate([np.arange(40), 301 + np.arange(32), 600 + np.arange(100)]), loud=loud)
    s.check()
    s.check(causal=False)


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("what", [np.inf, np.nan])
def test_values_that_are_no_numbers(km, gpu, kind, dim, what):
    """They come to the rows that see them and to no other."""
    rng = np.random.default_rng(dim + 2)
    for token, channel in ((200, 5), (299, dim - 1), (250, 0)):
        s = batch(km, rng, dim, kind)
        s.v[token, 1, channel] = what
        got, _ = s.check()
        assert np.isfinite(got[:, 0]).all() and np.isfinite(got[:token, 1]).all() and (~np.isfinite(got[token:300, 1])).any() and np.isfinite(got[300:]).all()
