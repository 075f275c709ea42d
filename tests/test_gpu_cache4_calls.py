"""Calls around the kernels of the 4-bit cache: bounds that say little, work space, recordings (-m gpu)."""
import numpy as np
import pytest

from test_gpu_cache4 import BF16, F16, Cache, Queries, bound_all, choice, device, select, to_bits
from test_zz_no_alloc import device_memory_in_use

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


def test_reserved_for_a_batch_and_smaller_ones(km, gpu):
    """A serving loop whose sequences end one after the other: reserved for the full batch, no smaller one allocates, and each can be recorded. (The full batch itself
    needs nothing: fewer units are taken in more parts.)"""
    rng = np.random.default_rng(3)
    heads, group, dim, page = 8, 2, 64, 16
    c = Cache(km, rng, heads, dim, page, 64 * 125 + 2, garbage=0x2B)  # (some numbers everywhere)
    kept = []
    for sequences, queries, length in ((64, 1, 2000), (63, 1, 2000), (40, 1, 1999), (7, 1, 2000), (1, 1, 600), (2, 40, 2000), (1, 64, 700), (5, 33, 1200)):
        s = Queries(km, rng, c, [length] * sequences, [queries] * sequences, group, BF16)
        s.bits, s.out = device(km, to_bits(s.q, BF16)), km.DeviceBuffer(2 * s.tokens * heads * group * dim)
        s.chosen, s.sparse = km.DeviceBuffer(4 * s.tokens * heads * 9), km.DeviceBuffer(2 * s.tokens * heads * group * dim)
        kept.append(s)
    bound_pages = np.arange(c.pages, dtype=np.int32)
    c.dev.bound(device(km, bound_pages), device(km, np.full(c.pages, page, np.int32)), c.pages)

    def step(s):
        c.dev.attend(s.batch, BF16, s.bits, s.out, s.scale)
        c.dev.select(s.batch, BF16, s.bits, s.chosen, 9)
        c.dev.attend(s.batch, BF16, s.bits, s.sparse, s.scale, chosen=s.chosen, top=9)

    def results(s):
        km.sync()
        return [b.read(np.uint16, b.nbytes // 2) for b in (s.out, s.sparse)]

    for s in kept:
        step(s)  # (the code is on the device)
    want = [results(s) for s in kept]
    km.check(km.hip_lib().kmx_shutdown())  # and the work space is not
    large = km.Cache4Batch(64, heads * group, 80 * 2, 64, 2000, device(km, np.int32([0])), device(km, np.int32([0])), device(km, np.int32([0])), kept[0].table.shape[1])
    c.dev.reserve(large, 9)
    km.sync()
    before = device_memory_in_use()
    for s, w in zip(kept, want):
        step(s)
        assert all(np.array_equal(a, b) for a, b in zip(results(s), w))
    assert device_memory_in_use() == before
    for s, w in zip(kept, want):
        with km.Graph() as g:
            step(s)
        for _ in range(3):
            for b in (s.out, s.sparse):
                b.zero()
            g.launch()
            assert all(np.array_equal(a, b) for a, b in zip(results(s), w))
            step(s)
        g.destroy()


def test_recordings_outlive_the_work_space(km, gpu):
    """Recorded attention, in parts of 16 rows and of 256, and the choice in two kernels: then the work space moves (a larger call) and goes (kmx_shutdown), and the
    replays are still the calls themselves."""
    rng = np.random.default_rng(5)
    c = Cache(km, rng, 1, 64, 16, 2500, garbage=0x2B)  # (some numbers everywhere)
    few = Queries(km, rng, c, [14000, 9000], [1, 2], 4, BF16)
    many = Queries(km, rng, c, [9000], [40], 2, BF16)
    large = Queries(km, rng, c, [15000], [600], 2, BF16)
    pages = np.arange(c.pages, dtype=np.int32)
    c.dev.bound(device(km, pages), device(km, np.full(c.pages, 16, np.int32)), c.pages)
    for s in (few, many, large):
        s.bits, s.out = device(km, to_bits(s.q, BF16)), km.DeviceBuffer(2 * s.tokens * s.group * 64)
    chosen, sparse = km.DeviceBuffer(4 * few.tokens * 12), km.DeviceBuffer(2 * few.tokens * 4 * 64)

    def step():
        c.dev.attend(few.batch, BF16, few.bits, few.out, few.scale)
        c.dev.attend(many.batch, BF16, many.bits, many.out, many.scale)
        c.dev.select(few.batch, BF16, few.bits, chosen, 12)
        c.dev.attend(few.batch, BF16, few.bits, sparse, few.scale, chosen=chosen, top=12)

    buffers = (few.out, many.out, chosen, sparse)

    def results():
        km.sync()
        return [b.read(np.uint16, b.nbytes // 2) for b in buffers]

    step()
    want = results()
    with km.Graph() as g:
        step()

    def replay():
        for b in buffers:
            b.zero()
        g.launch()
        assert all(np.array_equal(a, b) for a, b in zip(results(), want))

    replay()
    c.dev.attend(large.batch, BF16, large.bits, large.out, large.scale)  # more work space
    step()
    assert all(np.array_equal(a, b) for a, b in zip(results(), want))
    for _ in range(2):
        replay()
    km.check(km.hip_lib().kmx_shutdown())
    filler = [km.DeviceBuffer(1 << 22) for _ in range(4)]  # (where the work space was, for all one knows)
    for b in filler:
        b.write(np.full(1 << 20, 0x7FC00001, np.uint32))
    replay()
    km.sync()
    for b in filler:
        assert (b.read(np.uint32, 1 << 20) == 0x7FC00001).all()
    c.dev.attend(large.batch, BF16, large.bits, large.out, large.scale)
    replay()
    step()
    assert all(np.array_equal(a, b) for a, b in zip(results(), want))
    g.destroy()


def test_chosen_pages_behind_the_sequence(km, gpu):
    """Columns of the table behind a sequence's last page are left out wherever they are, also where their tokens' places would pass 32 bits."""
    rng = np.random.default_rng(6)
    c = Cache(km, rng, 1, 32, 256, 4)
    s = Queries(km, rng, c, [1000], [1], 2, BF16).fill(rng)
    pages, width = s.table[0, :4], (1 << 24) + 8
    table = np.full(width, -1, np.int32)
    table[:4] = pages
    table[[4, 5, 1 << 22, 1 << 23, (1 << 23) + 1, 1 << 24, (1 << 24) + 3]] = pages[0]
    s.table = table[None]
    s.batch = km.Cache4Batch(1, 2, 1, 1, 1000, device(km, s.starts), device(km, np.int32([1000])), device(km, table), width)
    for chosen in ([1, 4, 5, 1 << 22], [2, 1 << 23, (1 << 23) + 1, 1 << 24], [1 << 24, (1 << 24) + 3, -1, -1], [0, 1, 3, (1 << 24) + 7]):
        s.check(chosen=np.array(chosen)[None, None])


def test_levels_learned_from_rows_with_unusual_numbers(km, gpu):
    """Groups of 32 with infinities, NaN or nothing but zeros teach nothing: the levels are those of the other groups."""
    rng = np.random.default_rng(7)
    rows = rng.standard_t(6, size=(2000, 64)).astype(np.float32)
    want = km.cache4_learn_levels(rows)
    worse = np.concatenate([rows, rows[:300]])
    worse[2000:2100, [3, 40]], worse[2100:2200, [5, 63]], worse[2200:2300] = np.inf, np.nan, 0
    worse[2050, 7] = -np.inf
    assert np.array_equal(km.cache4_learn_levels(worse), want)
    for nothing in (np.full((4, 32), np.inf), np.full((4, 32), np.nan), np.zeros((4, 32))):
        with pytest.raises(ValueError):
            km.cache4_learn_levels(nothing)


def test_the_last_tile_that_31_bits_count(km, gpu):
    """A sequence of 2^31 - 1 tokens, all pages but the last the same: its last tokens hold all of the softmax, and queries before them do not see them."""
    rng = np.random.default_rng(8)
    c = Cache(km, rng, 1, 32, 256, 2)
    along = np.ones(32, np.float32)
    values = rng.normal(size=(512, 1, 32)).astype(np.float32)
    keys = np.zeros((512, 1, 32), np.float32)
    keys[256:] = 2 * np.arange(1, 257)[:, None, None] * along  # (held in 5 bits: some tokens in a row are alike, the next ones far above them)
    c.write(F16, keys, values, np.arange(512))
    length, counts, width = 2 ** 31 - 1, 100, 1 << 23
    table = np.zeros(width, np.int32)
    table[-1] = 1
    s = Queries(km, rng, c, [256], [counts], 1, F16)
    s.q = np.ones((counts, 1, 1, 32), np.float32)
    s.batch = km.Cache4Batch(1, 1, counts, counts, length, device(km, s.starts), device(km, np.int32([length])), device(km, table), width)
    got, lse = s.attend(scale=1.0)
    for i in range(counts):
        seen = slice(256, 256 + 256 - counts + i)  # of the last page, whose last token is not there
        k, v = c.k[seen, 0].astype(np.float64), c.v[seen, 0].astype(np.float64)
        score = k.sum(-1)
        p = np.exp(score - score.max())  # (e^-64 at most of what is not alike)
        want = p @ v / p.sum()
        assert np.all(np.abs(got[i, 0, 0] - want) <= 2.0 ** -11 * np.abs(want) + 2.0 ** -11 * (p @ np.abs(v)) / p.sum()), i
        assert abs(lse[i, 0, 0] - score.max() - np.log(p.sum())) <= 2.0 ** -20 * lse[i, 0, 0]
