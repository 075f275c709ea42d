"""Attention over the 4-bit cache where scores are far from zero, against its definition in 64 bits (-m gpu)."""
import numpy as np
import pytest

from test_gpu_cache4 import BF16, F16, UNIT, Cache, Queries

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("length,counts", [(150, 1), (150, 70), (9000, 1), (9000, 70)])  # few rows and many, in one part and in several
@pytest.mark.parametrize("kind,loud,scale", [(F16, 1e4, 1.0), (F16, 1e4, 1e3), (BF16, 1e8, 1.0), (BF16, 1e20, -1.0), (BF16, 1e30, 0.2), (BF16, 1e37, 1e3)])
def test_scores_far_from_zero(km, gpu, length, counts, kind, loud, scale):
    """Scores from thousands up to beyond what a float holds: the best token is all there is where the next one is behind it by more than scores
    may be off (products of `dim` terms and the score itself in 24 bits), and by 40 at least. The largest float stands for what is beyond it."""
    rng = np.random.default_rng(counts)
    c = Cache(km, rng, 1, 64, 64, -(-length // 64) + 1)
    s = Queries(km, rng, c, [length], [counts], 2, kind, loud=loud).fill(rng)
    got, lse = s.attend(scale=scale)
    assert np.isfinite(got).all() and not np.isnan(lse).any()
    at = np.arange(length)
    slots = s.table[0, at // 64] * 64 + at % 64
    k, v = c.k[slots, 0].astype(np.float64), c.v[slots, 0].astype(np.float64)
    clear = 0
    for i in range(counts):
        n = s.sees(0, i)
        q = s.q[i, 0].astype(np.float64)
        score = scale * q @ k[:n].T
        off = ((c.dim + 16) * 2.0 ** -23 * (abs(scale) * np.abs(q) @ np.abs(k[:n]).T).max(-1) + 2.0 ** -22 * np.abs(score).max(-1))
        best = score.argmax(-1)
        second = np.sort(score, -1)[:, -2] if n > 1 else np.full(2, -np.inf)
        for g in range(2):
            top = score[g, best[g]]
            if top - second[g] < 40 + 2 * off[g]:
                continue
            clear += 1
            assert np.all(np.abs(got[i, 0, g] - v[best[g]]) <= UNIT[kind] * np.abs(v[best[g]]) + 2.0 ** -11 * np.abs(v[best[g]])), (i, g)
            if loud < 1e30:
                assert abs(lse[i, 0, g] - top) <= off[g] + 2.0 ** -21 * abs(top)
            else:
                assert lse[i, 0, g] > 1e29
    assert clear >= counts  # half of the rows at least
