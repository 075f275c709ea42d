"""Attention over prompts with scores far from zero (csrc/prompt_attend_impl.h): masks of the type's lowest value, and scores of which only equal ones share a row (-m gpu)."""
import numpy as np
import pytest

from test_gpu_cache4 import BF16, F16, UNIT, from_bits, to_bits
from test_gpu_prompt import Prompts
from test_gpu_prompt_masks import Masked

pytestmark = pytest.mark.gpu

LOWEST = {BF16: float(from_bits(np.uint16([0xFF7F]), BF16)[0]), F16: -65504.0}


class LowestMask(Masked):
    """Hidden tokens have the lowest number of the type as a bias, times 1, or in half precision times the largest: below every other score by so much that they have no weight beside one."""

    def __init__(self, km, rng, heads, group, dim, counts, lengths, kind, hidden, **other):
        super().__init__(km, rng, heads, group, dim, counts, lengths, kind, hidden, **other)
        self.q[..., 0] = 1.0 if kind == BF16 else 65504.0
        self.k[..., 0] = np.where(self.hidden, LOWEST[kind], 0)

    def check_masked(self, causal=True, **how):
        """Rows that see others as if the masked ones were not there; rows that see masked ones only are some mean of their values, with the lse of their score."""
        got, lse = self.attend(causal, **how)
        want, want_lse, off, lse_off = self.expected(causal)
        for s, (nq, n) in enumerate(zip(self.counts, self.lengths)):
            for i in range(nq):
                t, sees = self.query_starts[s] + i, (max(0, n - nq + i + 1) if causal else n)
                for h in range(self.heads):
                    at = slice(self.token_starts[s], self.token_starts[s] + sees)
                    if not sees:
                        assert not got[t, h].any() and np.isneginf(lse[t, h]).all()
                    elif self.hidden[at, h].all():
                        v = self.v[at, h]
                        slack = (2 * UNIT[self.kind] + (sees + 64) * 2.0 ** -24) * np.abs(v).max(0) + 2.0 ** -25
                        assert np.all(got[t, h] <= v.max(0) + slack) and np.all(got[t, h] >= v.min(0) - slack), (t, h)
                        score = self.scale * self.q[t, h, :, 0].astype(np.float64) * LOWEST[self.kind]
                        assert np.all(np.abs(lse[t, h] - score) <= 2.0 ** -18 * np.abs(score)), (t, h)
                    else:
                        assert np.all(np.abs(got[t, h] - want[t, h]) <= off[t, h]) and np.all(np.abs(lse[t, h] - want_lse[t, h]) <= lse_off[t, h]), (t, h)


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("masked", [5, 32, 70])
def test_padding_in_front_by_the_lowest_value(km, gpu, kind, causal, dim, masked):
    rng = np.random.default_rng(dim + masked)
    LowestMask(km, rng, 1, 3, dim, [50, 96], [130, 96], kind, np.concatenate([np.arange(masked), 130 + np.arange(min(masked, 60))])).check_masked(causal)


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("heads,group,dim,counts,lengths", [(1, 2, 64, [3], [3000]), (2, 4, 128, [1, 1], [2900, 700]), (1, 1, 192, [40], [2048]), (1, 2, 256, [5], [2000])])
def test_masks_by_the_lowest_value_in_parts(km, gpu, kind, heads, group, dim, counts, lengths):
    rng = np.random.default_rng(dim)
    n = sum(lengths)
    for hidden in (np.arange(32), np.arange(n // 2), np.nonzero(np.repeat(rng.random(n // 32 + 1) < 0.6, 32)[:n])[0], np.setdiff1d(np.arange(n), [n - 150])):
        LowestMask(km, rng, heads, group, dim, counts, lengths, kind, hidden).check_masked()


@pytest.mark.parametrize("kind,power", [(F16, 22), (F16, 30), (BF16, 22), (BF16, 30), (BF16, 34), (BF16, 60), (BF16, 120)])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("dim,counts,lengths", [(32, [40], [300]), (64, [70, 3], [100, 33]), (128, [50], [200]), (192, [40], [90]), (256, [33], [100]), (64, [2], [3000])])
def test_equal_scores_far_from_zero(km, gpu, kind, power, sign, dim, counts, lengths):
    """Scores sign 2^power + n 2^(power - 22), n < 4, sums of exact products: tokens of a row's largest n share it, in the proportions that differences of scores say."""
    rng = np.random.default_rng(power + dim)
    s = Prompts(km, rng, 1, 2, dim, counts, lengths, kind)
    s.q[:], s.k[:] = 0, 0
    half = power // 2 if kind == F16 else power // 2 + (power - 22) % 2
    s.q[..., 0], s.k[..., 0] = 2.0 ** half, sign * 2.0 ** (power - half)
    n = rng.integers(0, 4, s.tokens)
    n[:50] = 0  # rises later
    step = power - 22
    s.q[..., 1], s.k[..., 1] = 2.0 ** (step // 2), n[:, None] * 2.0 ** (step - step // 2)
    assert np.array_equal(s.q, from_bits(to_bits(s.q, kind), kind)) and np.array_equal(s.k, from_bits(to_bits(s.k, kind), kind))
    for causal in (True, False):
        got, lse = s.attend(causal, scale=1.0)
        for b, (nq, m) in enumerate(zip(counts, lengths)):
            for i in range(nq):
                t, sees = s.query_starts[b] + i, (m - nq + i + 1 if causal else m)
                at = slice(s.token_starts[b], s.token_starts[b] + sees)
                v, steps = s.v[at, 0].astype(np.float64), n[at].astype(np.float64)
                p = np.exp((steps - steps.max()) * 2.0 ** step)
                want, size = p @ v / p.sum(), p @ np.abs(v) / p.sum()
                # the difference of two scores is exact, its product with log2 e is 3 2^step (1 + 2^-23) at most where it counts; then as always
                off = UNIT[kind] * np.abs(want) + (UNIT[kind] + 2.0 ** -18 + 2 * (sees + 64) * 2.0 ** -24) * size + (2.0 ** -25 + 2.0 ** -32 * m) * np.abs(v).max()
                assert np.all(np.abs(got[t, 0] - want) <= off), (t, causal, (np.abs(got[t, 0] - want) / off).max())
                top = sign * 2.0 ** power + steps.max() * 2.0 ** step
                assert np.all(np.abs(lse[t, 0] - (top + np.log(p.sum()))) <= 2.0 ** -21 * abs(top))


@pytest.mark.parametrize("kind,loud", [(BF16, 2.0 ** 40), (F16, 2.0 ** 13)])
@pytest.mark.parametrize("dim,counts,lengths", [(64, [100, 40], [300, 40]), (128, [70], [500]), (256, [40], [200]), (192, [3], [2500])])
def test_rows_far_from_zero_beside_others(km, gpu, kind, loud, dim, counts, lengths):
    """Every third query is so loud that its scores are far from zero: the others of its wavefront stay within the bounds that they have without it."""
    rng = np.random.default_rng(dim)
    s = Prompts(km, rng, 1, 2, dim, counts, lengths, kind)
    s.q[::3] = from_bits(to_bits(s.q[::3] * loud, kind), kind)
    got, lse = s.check(scale=1.0 if kind == F16 else None)
    assert np.isfinite(got).all() and np.isfinite(lse).all()


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("token", [0, 31, 40, 79])
def test_scores_of_plus_infinity(km, gpu, kind, token):
    """A softmax over them is no number: rows that see one are NaN, and no others."""
    rng = np.random.default_rng(5)
    s = Prompts(km, rng, 1, 2, 64, [80], [80], kind)
    s.q[..., 0] = 1
    s.k[token, 0, 0] = np.inf
    got, lse = s.attend()
    assert np.isfinite(got[:token]).all() and np.isfinite(lse[:token]).all() and np.isnan(got[token:]).all() and not np.isfinite(lse[token:]).any()
