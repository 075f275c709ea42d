"""The choice of pages over bounds that nobody made, and in the kernels that few sizes reach, against its definition in numpy (-m gpu)."""
import numpy as np
import pytest

from test_gpu_cache4 import BF16, F16, Cache, Queries, bound_all, choice, kept_bounds, select

pytestmark = pytest.mark.gpu

LARGEST = np.finfo(np.float32).max


def choice_by_kept_bounds(s, top, first, last, causal=True):
    """What is to be chosen by the bounds that lie on the device, whatever they are; a score is held to the finite numbers, NaN to the lowest."""
    c = s.c
    eight, scales = kept_bounds(c)
    out = np.full((s.tokens, c.heads, top), -1, np.int64)
    for b in range(len(s.lengths)):
        for i in range(s.counts[b]):
            t, n = s.starts[b] + i, -(-s.sees(b, i, causal) // c.page)
            pages = s.table[b, :n]
            known = (pages >= 0) & (pages < c.pages)
            at = np.where(known, pages, 0)
            for h in range(c.heads):
                q = s.q[t, h]
                m = np.abs(q).max()
                by = np.float32(1) / np.float32(m) * np.float32(127) if m > 0 else np.float32(0)
                q8 = np.clip(np.rint(q * by), -127, 127).astype(np.float64)  # (whole numbers below 2^24: exact)
                hi, lo = eight[at, h, :c.dim].astype(np.float64), eight[at, h, c.dim:].astype(np.float64)
                best = (np.maximum(q8, 0) @ hi.T + np.minimum(q8, 0) @ lo.T).max(0).astype(np.float32)
                with np.errstate(over="ignore", invalid="ignore"):
                    score = best * scales[at, h]
                score = np.where(np.isnan(score), -LARGEST, np.clip(score, -LARGEST, LARGEST))
                score = np.where(known, score, -np.inf)
                order = np.arange(n)
                score[(order < first) | (order + last >= n)] = np.inf
                best = np.sort(np.argsort(-score, kind="stable")[:top])
                out[t, h, :len(best)] = best
    return out


def put_scales(c, scales):
    """Other scales of all pages and heads, behind bounds that stay."""
    n = c.pages * c.heads
    raw = c.bounds.read(np.uint8, n * (2 * c.dim + 4))
    raw[n * 2 * c.dim:] = np.ascontiguousarray(scales, np.float32).reshape(-1).view(np.uint8)
    c.bounds.write(raw)


@pytest.mark.parametrize("heads,group,dim,page,lengths,counts,top,first,last", [
    (2, 4, 64, 16, [600, 40], [2, 1], 6, 1, 2), (1, 2, 96, 16, [9000], [3], 9, 2, 1),         # one kernel, few and more pages
    (1, 3, 32, 16, [13000, 400], [2, 3], 16, 1, 1), (1, 1, 32, 16, [140000], [1], 5, 2, 2)])  # two kernels, keys in LDS and in memory
@pytest.mark.parametrize("what", ["large", "infinite", "nan", "negative", "mixed", "some", "bytes"])
def test_bounds_that_nobody_made(km, gpu, heads, group, dim, page, lengths, counts, top, first, last, what):
    """Every entry is written, nothing behind the lists, the pages that are always taken are there, and the others by their scores as far as they have one."""
    rng = np.random.default_rng(dim + len(lengths))
    c = Cache(km, rng, heads, dim, page, sum(-(-n // page) for n in lengths) + 2)
    s = Queries(km, rng, c, lengths, counts, group, BF16)
    shape = (c.pages, c.heads)
    size = c.pages * c.heads * (2 * dim + 4)
    c.bounds.write(rng.integers(0, 256, size, dtype=np.uint8))
    unusual = np.float32([1e38, np.inf, np.nan, -np.nan, -np.inf, -1e38, LARGEST, 3e33, 0, -0.0, 1e-45])
    if what == "some":
        put_scales(c, np.where(rng.random(shape) < 0.3, rng.choice(unusual, shape), rng.random(shape)))
    elif what != "bytes":
        put_scales(c, {"large": np.full(shape, 1e38), "infinite": np.full(shape, np.inf), "nan": np.full(shape, np.nan), "negative": np.full(shape, -np.inf),
                       "mixed": rng.choice(unusual, shape)}[what])
    chosen = select(s, top, first, last)  # (nothing behind the lists: checked there)
    assert np.array_equal(chosen, choice_by_kept_bounds(s, top, first, last))
    for b, n in enumerate(lengths):
        for i in range(counts[b]):
            seen = -(-s.sees(b, i) // page)
            for h in range(heads):
                assert set(range(min(first, seen))) | set(range(max(0, seen - last), seen)) <= set(chosen[s.starts[b] + i, h].tolist())


@pytest.mark.parametrize("heads,group,dim,page,lengths,counts,top,first,last", [
    (1, 4, 160, 16, [9700], [3], 9, 1, 1), (1, 2, 256, 16, [12200, 8300], [2, 1], 12, 1, 1), (1, 20, 192, 16, [10000], [1], 6, 0, 1),  # one kernel of 8 wavefronts, two tiles of pages each
    (1, 4, 128, 16, [13000, 12400], [20, 7], 10, 1, 1), (2, 2, 64, 16, [12500], [17], 5, 1, 0), (1, 16, 256, 16, [12900], [3], 8, 1, 1),  # two kernels, several tiles of queries
    (1, 1, 32, 16, [140000], [2], 700, 1, 1)])                                                                                          # keys from memory
def test_choice_in_kernels_that_few_sizes_reach(km, gpu, heads, group, dim, page, lengths, counts, top, first, last):
    rng = np.random.default_rng(dim + heads)
    c = Cache(km, rng, heads, dim, page, sum(-(-n // page) for n in lengths) + 2)
    s = Queries(km, rng, c, lengths, counts, group, F16).fill(rng)
    want = bound_all(s)
    chosen = select(s, top, first, last)
    assert np.array_equal(chosen, choice_by_kept_bounds(s, top, first, last))
    if max(lengths) < 20000:  # (the definition page by page takes long)
        assert np.array_equal(chosen, choice(s, want, top, first, last, True))
    s.check(chosen=chosen)
    apart = select(s, top, first, last, causal=False)
    assert np.array_equal(apart, choice_by_kept_bounds(s, top, first, last, causal=False))
