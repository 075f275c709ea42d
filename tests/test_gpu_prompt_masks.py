"""Attention over prompts with tokens whose score is minus infinity (csrc/prompt_attend_impl.h): a channel of the keys that masks them out, against the softmax over the others in 64 bits
(-m gpu)."""
import numpy as np
import pytest

from test_gpu_cache4 import BF16, F16, UNIT, from_bits, to_bits
from test_gpu_prompt import Prompts

pytestmark = pytest.mark.gpu


class Masked(Prompts):
    """Prompts whose first channel is a bias: `hidden` tokens of a head have a key there that makes every score of theirs minus infinity."""

    def __init__(self, km, rng, heads, group, dim, counts, lengths, kind, hidden, how="infinite", **other):
        super().__init__(km, rng, heads, group, dim, counts, lengths, kind, **other)
        self.hidden = np.zeros((self.tokens, heads), bool)
        self.hidden[hidden] = True
        bias, key = {"infinite": (1.0, -np.inf), "overflow": (2.0 ** 100, -2.0 ** 100)}[how]  # (products of bfloat16 numbers below the smallest float)
        self.q[..., 0] = bias
        self.k[..., 0] = np.where(self.hidden, key, 0)

    def expected(self, causal=True, scale=None):
        """As Prompts.expected, with the same bounds, over the tokens that are seen and not hidden: the others have no weight at all."""
        scale = self.scale if scale is None else scale
        shape = (self.queries, self.heads, self.group)
        out, lse = np.zeros(shape + (self.dim,)), np.full(shape, -np.inf)
        off, lse_off = np.zeros_like(out), np.zeros(shape)
        for s, (nq, n) in enumerate(zip(self.counts, self.lengths)):
            rows, at = slice(self.query_starts[s], self.query_starts[s] + nq), slice(self.token_starts[s], self.token_starts[s] + n)
            sees = np.maximum(0, n - nq + 1 + np.arange(nq)) if causal else np.full(nq, n)
            for h in range(self.heads):
                k, v = np.where(self.hidden[at, h, None], 0, self.k[at, h]).astype(np.float64), self.v[at, h].astype(np.float64)
                seen = (np.arange(n) < sees[:, None]) & ~self.hidden[at, h]
                some = seen.any(-1)
                for g in range(self.group):
                    if not some.any():
                        continue
                    q = self.q[rows, h, g].astype(np.float64)
                    score = np.where(seen, scale * q @ k.T, -np.inf)
                    top = np.where(some, score.max(-1), 0)[:, None]
                    p = np.where(seen, np.exp(score - top), 0)
                    total = np.maximum(p.sum(-1, keepdims=True), 1e-300)
                    o, size = p @ v / total, p @ np.abs(v) / total
                    length = np.abs(score, where=seen, out=np.zeros_like(score))
                    delta = ((self.dim + 16) * 2.0 ** -23 * (abs(scale) * np.abs(q) @ np.abs(k).T).max(-1) + 2.0 ** -22 * length.max(-1))[:, None]
                    terms = (sees[:, None] + 64) * 2.0 ** -24
                    out[rows, h, g] = np.where(some[:, None], o, 0)
                    lse[rows, h, g] = np.where(some, top[:, 0] + np.log(total[:, 0]), -np.inf)
                    off[rows, h, g] = UNIT[self.kind] * np.abs(o) + (UNIT[self.kind] + 2 * delta + 2 * terms) * size + (2.0 ** -25 + 2.0 ** -32 * n) * np.abs(v).max(initial=0)
                    lse_off[rows, h, g] = (delta + terms)[:, 0] + 2.0 ** -21 * (1 + np.abs(np.where(some, lse[rows, h, g], 0)))
        return out, lse, off, lse_off


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("masked", [32, 33, 64, 100])
def test_padding_in_front(km, gpu, kind, causal, dim, masked):
    """The first tiles have no weight; rows that see nothing else are zeros and minus infinity."""
    rng = np.random.default_rng(dim + masked)
    Masked(km, rng, 1, 3, dim, [50, 96], [130, 96], kind, np.concatenate([np.arange(masked), 130 + np.arange(min(masked, 70))])).check(causal)


@pytest.mark.parametrize("kind,how", [(F16, "infinite"), (BF16, "infinite"), (BF16, "overflow")])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_a_row_that_rises_later_beside_rows_that_do_not(km, gpu, kind, how, dim):
    """What the other rows of the wavefront have added up by then stays."""
    rng = np.random.default_rng(dim)
    for row, token in ((5, 80), (31, 70), (0, 95)):
        s = Masked(km, rng, 1, 1, dim, [40], [96], kind, np.arange(32), how)
        with np.errstate(all="ignore"):
            s.k[token, 0, 1:] = from_bits(to_bits(s.q[row, 0, 0, 1:] * 3.0, kind), kind)
        s.check(causal=False)
        s.check()


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("low", [-150.0, -1000.0, -10000.0])
def test_scores_far_below_zero_behind_masked_ones(km, gpu, kind, low):
    rng = np.random.default_rng(3)
    s = Masked(km, rng, 1, 2, 64, [70], [160], kind, np.arange(40))
    s.q[..., 1] = 8
    s.k[..., 1] = from_bits(to_bits(np.float32([low]), kind), kind)
    s.check()
    s.check(causal=False)


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("what", ["first", "half", "blocks", "all but one"])
@pytest.mark.parametrize("heads,group,dim,counts,lengths", [(1, 2, 64, [3], [3000]), (2, 4, 128, [1, 1], [2900, 700]), (1, 1, 192, [40], [2048]), (1, 2, 256, [5], [2000])])
def test_masked_tokens_in_parts(km, gpu, kind, what, heads, group, dim, counts, lengths):
    """Parts that begin with masked tokens, or have no others."""
    rng = np.random.default_rng(dim + len(what))
    n = sum(lengths)
    hidden = {"first": np.arange(32), "half": np.arange(n // 2), "blocks": np.nonzero(np.repeat(rng.random(n // 32 + 1) < 0.6, 32)[:n])[0], "all but one": np.setdiff1d(np.arange(n), [n - 150])}[what]
    s = Masked(km, rng, heads, group, dim, counts, lengths, kind, hidden)
    first = s.check()
    again = s.check(gaps=(1, 0), key_gaps=(0, 1), out_gaps=(1, 1), offset=1)
    assert np.array_equal(first[0], again[0]) and np.array_equal(first[1], again[1])


@pytest.mark.parametrize("kind", [F16, BF16])
def test_masked_tokens_of_one_head_and_of_none_left(km, gpu, kind):
    rng = np.random.default_rng(4)
    s = Masked(km, rng, 2, 2, 64, [90], [90], kind, [])
    s.hidden[:, 1] = True
    s.k[:, 1, 0] = -np.inf
    got, lse = s.check()
    assert not got[:, 1].any() and np.isneginf(lse[:, 1]).all() and np.isfinite(lse[:, 0]).all()
