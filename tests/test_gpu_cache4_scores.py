"""Attention over the 4-bit cache where scores are far from zero or far apart and where rows are small, against its definition in 64 bits (-m gpu)."""
import numpy as np
import pytest

from test_gpu_cache4 import BF16, F16, F32, UNIT, Cache, Queries, device, from_bits, to_bits

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


SEQUENCES, TOKENS = 128, 65536


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("queries", [1, 17])  # 16 rows and 256 a work-group, all tokens in one part
@pytest.mark.parametrize("behind", [12.0, 15.0, 17.4])
def test_one_token_far_above_the_others(km, gpu, kind, queries, behind):
    """One token holds nearly all of the softmax and has a value of zero: what all the others add up to is the result. Off by the roundings of the type, of a
    probability (2^-11 of it, 2^-40 at least), of scores and of sums in 24 bits."""
    rng = np.random.default_rng(queries)
    heads, group, dim, page = 4, 4, 32, 256
    c = Cache(km, rng, heads, dim, page, TOKENS // page)
    along = np.where(rng.random(dim) < 0.5, -1.0, 1.0)
    scale = 1 / np.sqrt(dim)
    keys, values = 0.3 * rng.normal(size=(TOKENS, heads, dim)), 1 + 0.3 * rng.normal(size=(TOKENS, heads, dim))
    sink = 1000
    keys[sink], values[sink] = along * behind / (scale * dim), 0
    c.write(F16, np.float32(keys), np.float32(values), np.arange(TOKENS))
    one = Queries(km, rng, c, [TOKENS], [queries], group, kind)  # (its table is replaced: all sequences look at the same pages in order)
    one.table = np.arange(TOKENS // page, dtype=np.int32)[None]
    q = np.float32(along + 0.1 * rng.normal(size=(queries, heads, group, dim)))
    s = Queries(km, rng, c, [0] * SEQUENCES, [queries] * SEQUENCES, group, kind)
    s.q = np.tile(q.astype(np.float16).astype(np.float32) if kind == F16 else (q.view(np.uint32) & 0xFFFF0000).view(np.float32), (SEQUENCES, 1, 1, 1))
    table = np.tile(one.table, (SEQUENCES, 1))
    s.batch = km.Cache4Batch(SEQUENCES, heads * group, SEQUENCES * queries, queries, TOKENS, device(km, s.starts), device(km, np.full(SEQUENCES, TOKENS, np.int32)),
                             device(km, table), table.shape[1])
    got, lse = s.attend()
    assert np.array_equal(got, np.tile(got[:queries], (SEQUENCES, 1, 1, 1))) and np.array_equal(lse, np.tile(lse[:queries], (SEQUENCES, 1, 1)))
    for i in range(queries):
        n = TOKENS - queries + i + 1
        for h in range(heads):
            k, v = c.k[:n, h].astype(np.float64), c.v[:n, h].astype(np.float64)
            x = s.q[i, h].astype(np.float64)
            score = scale * x @ k.T
            top = score.max(-1, keepdims=True)
            p = np.exp(score - top)
            assert np.all(p.argmax(-1) == sink)
            total = p.sum(-1, keepdims=True)
            want = p @ v / total
            delta = ((dim + 16) * 2.0 ** -23 * (scale * np.abs(x) @ np.abs(k).T).max(-1) + 2.0 ** -22 * np.abs(score).max(-1))[:, None]
            terms = (n + 64) * 2.0 ** -24
            off = UNIT[kind] * np.abs(want) + (2.0 ** -11 + 2 * delta + 2 * terms) * (p @ np.abs(v) / total) + n * 2.0 ** -40 * np.abs(v).max() / total
            assert np.all(np.abs(got[i, h] - want) <= off), (np.abs(got[i, h] - want) / off).max()
            assert np.all(np.abs(lse[i, h] - (top + np.log(total))[:, 0]) <= delta[:, 0] + terms + 2.0 ** -21 * (1 + np.abs(lse[i, h])))


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("dim,counts", [(64, [1, 1]), (64, [70, 33]), (256, [1, 3])])
@pytest.mark.parametrize("size", [1e-3, 1e-4, 1e-6])
def test_small_rows(km, gpu, kind, dim, counts, size):
    """Numbers of the cache below 2^-14 are held in more places than half precision has: attention takes them rounded to it, which is what read returns as F16."""
    rng = np.random.default_rng(dim)
    c = Cache(km, rng, 1, dim, 32, 14)
    s = Queries(km, rng, c, [300, 90], counts, 2, kind)
    for b, n in enumerate(s.lengths):
        at = np.arange(n)
        c.write(F32, *(np.float32(size * rng.normal(size=(n, 1, dim))) for _ in range(2)), s.table[b, at // 32] * 32 + at % 32)
    everywhere = np.arange(14 * 32)
    k, v = (x.astype(np.float32) for x in c.read(F16, everywhere))
    written = np.zeros(14 * 32, bool)
    for b, n in enumerate(s.lengths):
        at = np.arange(n)
        written[s.table[b, at // 32] * 32 + at % 32] = True
    assert np.array_equal(k[written], c.k[written].astype(np.float16).astype(np.float32))
    assert np.array_equal(k[written], c.k[written]) == (size == 1e-3)  # (products of these levels and scales still fit there)
    c.k[written], c.v[written] = k[written], v[written]
    got, lse = s.attend(scale=1 / (size * np.sqrt(dim)))
    want, want_lse, off, lse_off = s.expected(scale=1 / (size * np.sqrt(dim)))
    if kind == F16:
        off = off + 2.0 ** -25  # results below 2^-14 have no more places either
    assert np.all(np.abs(got - want) <= off), (np.abs(got - want) / off).max()
    assert np.all(np.abs(lse - want_lse) <= lse_off)


@pytest.mark.parametrize("counts", [[1], [70]])
def test_queries_below_the_normal_numbers(km, gpu, counts):
    rng = np.random.default_rng(9)
    c = Cache(km, rng, 1, 64, 64, 5)
    s = Queries(km, rng, c, [150], counts, 2, BF16, loud=2.0 ** -126).fill(rng)
    small = from_bits(to_bits(s.q / 64, BF16), BF16)
    s.q = small
    assert np.abs(small).max() < 2.0 ** -126 and np.abs(small).max() > 0
    s.check(scale=2.0 ** 126)
