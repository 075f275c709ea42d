"""Attention weights added up (kmx_cache4_weigh) and eviction by them (kmx_cache4_evict) against their definitions: sums in 64 bits, choices and moves as whole numbers,
moved rows byte for byte (-m gpu)."""
import numpy as np
import pytest

from test_gpu_cache4 import BF16, F16, Cache, Queries, device, ordinary, to_bits

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- weights ------------------------

def weigh(s, weights, causal=True, scale=None, lse=None, offset=0, gaps=(0, 0)):
    """weights: host array, added to on the device."""
    km, c = s.km, s.c
    heads = c.heads * s.group
    qh = c.dim + gaps[0]
    qt = heads * qh + gaps[1]
    flat = np.full((s.tokens, qt), 3, np.float32)
    flat[:, :heads * qh].reshape(s.tokens, heads, qh)[:, :, :c.dim] = s.q.reshape(s.tokens, heads, c.dim)
    q = device(km, to_bits(np.concatenate([np.zeros(offset, np.float32), flat.reshape(-1)]), s.kind))
    w = device(km, weights)
    c.dev.weigh(s.batch, s.kind, km.DeviceView(q.ptr.value + 2 * offset, 0), device(km, np.float32(lse)), w, s.scale if scale is None else scale, causal=causal, q_token_stride=qt, q_head_stride=qh)
    km.sync()
    return w.read(np.float32, weights.size).reshape(weights.shape).astype(np.float64)


def weighed(s, weights, lse, causal=True, scale=None):
    """(weights, how far they may be off): scores with as many terms of 24 bits as a row has channels, exponents and sums of 24 bits."""
    c, scale = s.c, s.scale if scale is None else scale
    want, off = weights.astype(np.float64), np.zeros(weights.shape)
    for b, n in enumerate(s.lengths):
        at = np.arange(n)
        pages = s.table[b, at // c.page]
        there = (pages >= 0) & (pages < c.pages)
        slots = np.where(there, pages, 0) * c.page + at % c.page
        for i in range(s.counts[b]):
            t = s.starts[b] + i
            mask = there & (at < s.sees(b, i, causal))
            if not mask.any():
                continue
            for h in range(c.heads):
                k, q = c.k[slots[mask], h].astype(np.float64), s.q[t, h].astype(np.float64)
                score = scale * q @ k.T
                p = np.exp(score - lse[t, h][:, None])
                delta = (c.dim + 16) * 2.0 ** -23 * (abs(scale) * np.abs(q) @ np.abs(k).T) + 2.0 ** -22 * (np.abs(score) + np.abs(lse[t, h][:, None]) + 1)
                np.add.at(want, (pages[mask], h, at[mask] % c.page), p.sum(0))
                np.add.at(off, (pages[mask], h, at[mask] % c.page), (2 * p * delta).sum(0) + 1e-37)
    rows = max([1] + [n * s.group for n in s.counts])
    return want, off + 2.0 ** -23 * (rows + 4) * np.abs(want)


def check_weights(s, rng, causal=True, scale=None, **how):
    c = s.c
    weights = np.float32(rng.random((c.pages, c.heads, c.page)))
    lse = np.float32(s.expected(causal, scale=scale)[1]).astype(np.float64)
    got = weigh(s, weights, causal, scale, lse, **how)
    want, off = weighed(s, weights, lse, causal, scale)
    assert np.all(np.abs(got - want) <= off), (np.abs(got - want) / np.maximum(off, 1e-300)).max()
    added = (got - weights).sum()
    rows = sum(sum(1 for i in range(n) if s.sees(b, i, causal)) for b, n in enumerate(s.counts)) * s.group * c.heads
    assert abs(added - rows) <= 1e-4 * rows + weights.size * 2.0 ** -23  # the weights of a row are 1 together
    return got


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,group,dim,page,lengths,counts", [
    (1, 1, 32, 16, [1], [1]), (2, 4, 64, 32, [1, 15, 16, 17, 0, 63], [1] * 6), (2, 8, 128, 64, [64, 65, 257, 700], [1, 2, 3, 1]), (1, 17, 96, 256, [255, 513], [1, 4]),
    (3, 3, 160, 16, [200, 30], [25, 30]), (1, 2, 192, 128, [600], [40]), (2, 5, 224, 64, [77, 5], [1, 5]), (1, 3, 256, 64, [300, 3], [70, 1]), (1, 16, 64, 16, [130], [9])])
def test_weights_of_the_tokens(km, gpu, kind, causal, heads, group, dim, page, lengths, counts):
    rng = np.random.default_rng(dim + group)
    c = Cache(km, rng, heads, dim, page, sum(-(-n // page) for n in lengths) + 2)
    check_weights(Queries(km, rng, c, lengths, counts, group, kind).fill(rng), rng, causal)


def test_more_queries_than_tokens(km, gpu):
    rng = np.random.default_rng(1)
    c = Cache(km, rng, 2, 64, 16, 8)
    check_weights(Queries(km, rng, c, [2, 0, 1, 40], [4, 9, 2, 60], 2, F16).fill(rng), rng)


@pytest.mark.parametrize("scale", [0.0, -0.3, 3.0])
def test_weights_at_other_scales(km, gpu, scale):
    rng = np.random.default_rng(2)
    c = Cache(km, rng, 1, 64, 64, 5)
    check_weights(Queries(km, rng, c, [200], [3], 2, F16, loud=0.5).fill(rng), rng, scale=scale)


def test_weights_with_strides_and_odd_addresses(km, gpu):
    rng = np.random.default_rng(3)
    c = Cache(km, rng, 2, 96, 32, 10)
    s = Queries(km, rng, c, [100, 41], [3, 1], 3, BF16).fill(rng)
    for how in (dict(gaps=(8, 32), offset=8), dict(gaps=(1, 2), offset=1)):
        check_weights(s, np.random.default_rng(4), **how)


def test_weights_of_pages_that_are_shared_or_not_there(km, gpu):
    """Two sequences with a page of the same tokens: both add to it. Pages outside the cache get nothing, nor does anything else."""
    rng = np.random.default_rng(5)
    c = Cache(km, rng, 2, 64, 16, 12)
    s = Queries(km, rng, c, [40, 40, 64], [1, 1, 1], 2, BF16).fill(rng)
    s.table[1, :2] = s.table[0, :2]
    s.table[2, 1:3] = [-1, 1 << 20]
    s.batch = km.Cache4Batch(3, 4, 3, 1, 64, device(km, s.starts), device(km, np.int32(s.lengths)), device(km, s.table), s.table.shape[1])
    check_weights(s, rng)
    lse = s.expected()[1]
    lse[0, 0, 0] = np.nan
    weights = np.zeros((c.pages, 2, 16), np.float32)
    got = weigh(s, weights, lse=lse)
    nan = np.isnan(got)
    assert nan[s.table[0, :3], 0].sum() == 40 and nan.sum() == 40, "NaN stays with the tokens of its head that are seen"


def test_weights_recorded(km, gpu):
    rng = np.random.default_rng(6)
    c = Cache(km, rng, 2, 64, 64, 20)
    s = Queries(km, rng, c, [700, 300], [1, 1], 4, BF16).fill(rng)
    q, lse, w = device(km, to_bits(s.q, BF16)), device(km, np.float32(s.expected()[1])), device(km, np.zeros(20 * 2 * 64, np.float32))
    c.dev.weigh(s.batch, BF16, q, lse, w, s.scale)
    km.sync()
    want = w.read(np.float32, 20 * 2 * 64)
    with km.Graph() as g:
        c.dev.weigh(s.batch, BF16, q, lse, w, s.scale)
    total = want.copy()
    for _ in range(4):
        g.launch()
        km.sync()
        total += want
        assert np.array_equal(w.read(np.float32, 20 * 2 * 64), total)
        c.dev.weigh(s.batch, BF16, q, lse, w, s.scale)
        km.sync()
        total += want
        assert np.array_equal(w.read(np.float32, 20 * 2 * 64), total)
    g.destroy()


# ---------------------------------------------------------------- eviction -----------------------

def choice(w, n, keep, first, recent):
    """Where the tokens of the new places come from: weights w of the n tokens of a sequence and head."""
    if n <= keep:
        return list(range(n))
    edge = keep - recent
    key = [(-np.inf if np.isnan(w[t]) else float(w[t]), not np.isnan(w[t])) for t in range(n)]  # NaN below minus infinity
    best = sorted(range(first, n - recent), key=lambda t: (-key[t][0], not key[t][1], t))[:edge - first]
    stay = set(range(first)) | set(best)
    free = iter(sorted(t for t in stay if t >= edge))
    return [t if t in stay else next(free) for t in range(edge)] + list(range(n - recent, n))


class Evict:
    def __init__(self, km, rng, heads, dim, page, lengths, keep, first, recent, weights=None, extra=1, most=None):
        self.km, self.lengths, self.keep, self.first, self.recent = km, lengths, keep, first, recent
        self.c = c = Cache(km, rng, heads, dim, page, sum(-(-n // page) for n in lengths) + 3, garbage=0x2B)
        self.s = Queries(km, rng, c, lengths, [0] * len(lengths), 1, F16, extra=extra)
        self.raw = rng.integers(0, 256, c.blocks.nbytes, dtype=np.uint8)  # any bytes: rows move as they are
        c.blocks.write(self.raw)
        self.weights = np.exp(rng.normal(size=(c.pages, heads, page)) * 3).astype(np.float32) if weights is None else weights(c.pages, heads, page)
        self.w = device(km, self.weights)
        self.kept, self.left = device(km, np.full(len(lengths) * heads * max(1, keep), 77, np.int32)), device(km, np.full(len(lengths), 77, np.int32))
        self.batch = km.Cache4Batch(len(lengths), heads, 0, 0, max(lengths) if most is None else most, device(km, self.s.starts), device(km, np.int32(lengths)), device(km, self.s.table), self.s.table.shape[1])

    def rows(self, raw):
        """Where the bytes of each page, head and token lie: (pages, heads, page, bytes of a row)."""
        c, dim = self.c, self.c.dim
        b = raw.reshape(c.pages, c.heads, c.page // 16, 18 * dim)
        keys, values = b[..., :8 * dim].reshape(b.shape[:3] + (16, dim // 2)), b[..., 8 * dim:16 * dim].reshape(b.shape[:3] + (dim // 2, 16)).swapaxes(-1, -2)
        ks, vs = b[..., 16 * dim:17 * dim].reshape(b.shape[:3] + (16, dim // 16)), b[..., 17 * dim:].reshape(b.shape[:3] + (dim // 32, 16, 2)).swapaxes(-2, -3).reshape(b.shape[:3] + (16, dim // 16))
        return np.concatenate([keys, values, ks, vs], -1).reshape(c.pages, c.heads, c.page, -1)

    def call(self):
        self.c.dev.evict(self.batch, self.w, self.keep, self.first, self.recent, self.kept, self.left)

    def results(self):
        self.km.sync()
        c = self.c
        return (self.kept.read(np.int32, len(self.lengths) * c.heads * self.keep).reshape(len(self.lengths), c.heads, self.keep), self.left.read(np.int32, len(self.lengths)),
                self.w.read(np.float32, self.weights.size).reshape(self.weights.shape), self.rows(c.blocks.read(np.uint8, self.raw.size)))

    def expected(self):
        c = self.c
        kept = np.full((len(self.lengths), c.heads, self.keep), -1, np.int32)
        weights, rows, old = self.weights.copy(), self.rows(self.raw).copy(), self.rows(self.raw)
        for b, n in enumerate(self.lengths):
            pages = self.s.table[b]
            for h in range(c.heads):
                at = np.arange(n)
                w = self.weights[pages[at // c.page], h, at % c.page] if n else []
                new = choice(w, n, self.keep, self.first, self.recent)
                kept[b, h, :len(new)] = new
                if n <= self.keep:
                    continue
                to, fr = np.arange(self.keep), np.array(new, int)
                rows[pages[to // c.page], h, to % c.page] = old[pages[fr // c.page], h, fr % c.page]
                weights[pages[at // c.page], h, at % c.page] = 0
                weights[pages[to // c.page], h, to % c.page] = w[fr]
        return kept, np.minimum(self.lengths, self.keep), weights, rows

    def check(self):
        self.call()
        got, want = self.results(), self.expected()
        for name, a, b in zip(("left", "kept", "weights", "rows"), (got[1], got[0], got[2].view(np.uint32), got[3]), (want[1], want[0], want[2].view(np.uint32), want[3])):
            assert np.array_equal(a, b), (name, np.argwhere(np.asarray(a) != np.asarray(b))[:5])
        return got


@pytest.mark.parametrize("heads,dim,page,lengths,keep,first,recent", [
    (1, 32, 16, [20], 10, 0, 0), (2, 64, 32, [100, 40, 7, 0], 40, 4, 8), (3, 96, 64, [500, 129, 128], 128, 1, 64), (2, 128, 16, [300, 65], 64, 0, 64), (1, 160, 256, [1000], 999, 4, 100),
    (2, 192, 64, [700, 200], 150, 150, 0), (1, 224, 128, [400], 33, 1, 32), (2, 256, 64, [130, 300], 100, 2, 0), (4, 128, 64, [65, 66, 1025], 64, 4, 32), (1, 64, 16, [50, 51], 1, 0, 1),
    (2, 64, 64, [200, 90], 1, 1, 0), (1, 32, 16, [40], 17, 3, 5), (2, 64, 64, [5000, 2000, 100], 1500, 4, 1100)])
def test_sequences_back_to_their_budget(km, gpu, heads, dim, page, lengths, keep, first, recent):
    rng = np.random.default_rng(dim + keep)
    Evict(km, rng, heads, dim, page, lengths, keep, first, recent).check()


def test_nothing_is_kept_and_nothing_has_to_go(km, gpu):
    rng = np.random.default_rng(1)
    Evict(km, rng, 2, 64, 16, [50, 3], 0, 0, 0).check()
    Evict(km, rng, 2, 64, 16, [50, 3], 50, 4, 8).check()
    Evict(km, rng, 2, 64, 16, [50, 3], 70, 4, 8).check()


def some(kind, rng):
    def make(pages, heads, page):
        w = np.exp(rng.normal(size=(pages, heads, page)) * 3).astype(np.float32)
        if kind == "equal":
            w[:] = 0.25
        elif kind == "zeros":
            w[rng.random(w.shape) < 0.8] = 0
            w[rng.random(w.shape) < 0.3] *= -0.0
        elif kind == "few":
            w = rng.integers(0, 4, w.shape).astype(np.float32)
        elif kind == "anything":
            w = (w * rng.choice([-1, 1], w.shape)).astype(np.float32)
            for x in (np.nan, -np.nan, np.inf, -np.inf, 1e-45, -1e-45, 3.4e38, -3.4e38):
                w[rng.random(w.shape) < 0.07] = x
        elif kind == "nan":
            w[:] = np.nan
        return w
    return make


@pytest.mark.parametrize("kind", ["equal", "zeros", "few", "anything", "nan"])
@pytest.mark.parametrize("lengths,keep,first,recent", [([200, 130], 70, 4, 10), ([3000, 70], 1000, 0, 65), ([66], 65, 1, 1)])
def test_equal_weights_and_unusual_ones(km, gpu, kind, lengths, keep, first, recent):
    rng = np.random.default_rng(len(kind) + keep)
    Evict(km, rng, 2, 64, 16, lengths, keep, first, recent, weights=some(kind, rng)).check()


@pytest.mark.parametrize("length,keep,first,recent", [(24576, 10000, 0, 0), (40000, 30000, 4, 5000), (70001, 129, 1, 64), (30000, 29999, 4, 2000)])
def test_long_sequences(km, gpu, length, keep, first, recent):
    """More tokens than have their keys in LDS among them."""
    rng = np.random.default_rng(length)
    Evict(km, rng, 1, 32, 256, [length, 50], keep, first, recent).check()


def test_long_and_short_sequences_in_one_call(km, gpu):
    """Weights that stay in LDS beside others that are read again for every pass, and sequences that stay as they are."""
    rng = np.random.default_rng(21)
    e = Evict(km, rng, 2, 32, 64, [50000, 3000, 700, 12000, 1001], 1000, 4, 64)
    e.check()


def test_the_longest_sequences(km, gpu):
    rng = np.random.default_rng(7)
    e = Evict(km, rng, 1, 32, 256, [262144], 262000, 1000, 100)
    e.check()


def test_again_and_again(km, gpu):
    """A cache at its budget: a token more each time. The recent ones stay the last in their order, and what came first and is heavy never leaves."""
    rng = np.random.default_rng(8)
    e = Evict(km, rng, 2, 64, 16, [65, 65], 64, 2, 8)
    for step in range(12):
        e.weights = e.w.read(np.float32, e.weights.size).reshape(e.weights.shape)
        e.raw = e.c.blocks.read(np.uint8, e.raw.size)
        got = e.check()
        assert np.all(got[0][:, :, -8:] == np.arange(57, 65)) and np.all(got[0][:, :, :2] == np.arange(2))
        weights = got[2].copy()
        for b in range(2):  # the next token
            page = e.s.table[b, 64 // 16]
            assert np.all(weights[page, :, 0] == 0)
            weights[page, :, 0] = rng.random(2)
        e.w.write(weights)


def test_lengths_and_pages_that_are_not_there(km, gpu):
    """Lengths beyond the table or the bound are cut; tokens on pages outside the cache are the lightest, and what would move there or come from there stays away."""
    rng = np.random.default_rng(9)
    e = Evict(km, rng, 1, 64, 16, [100, 40], 30, 0, 4, most=90)
    e.lengths = [90, 40]
    e.check()
    e = Evict(km, rng, 1, 64, 16, [100], 30, 0, 4, extra=0)
    long = km.Cache4Batch(1, 1, 0, 0, 262144, device(km, np.int32([0, 0])), device(km, np.int32([1 << 30])), device(km, e.s.table), e.s.table.shape[1])
    e.c.dev.evict(long, e.w, 30, 0, 4, e.kept, e.left)
    got = e.results()
    at = np.arange(112)
    assert got[0][0, 0].tolist() == choice(e.weights[e.s.table[0, at // 16], 0, at % 16], 112, 30, 0, 4) and got[1][0] == 30
    e = Evict(km, rng, 1, 64, 16, [100, -7], 30, 0, 4)
    got = e.check() if False else (e.call(), e.results())[1]
    assert got[1].tolist() == [30, 0] and np.all(got[0][1] == -1)
    e = Evict(km, rng, 1, 64, 16, [100], 30, 0, 4)
    before = e.rows(e.raw)
    e.s.table[0, [1, 3]] = [-1, 1 << 20]
    e.batch = km.Cache4Batch(1, 1, 0, 0, 100, device(km, e.s.starts), device(km, np.int32([100])), device(km, e.s.table), e.s.table.shape[1])
    e.call()
    kept, left, weights, rows = e.results()
    w = np.array([np.nan if t // 16 in (1, 3) else e.weights[e.s.table[0, t // 16], 0, t % 16] for t in range(100)])
    assert kept[0, 0].tolist() == choice(w, 100, 30, 0, 4)
    page = e.s.table[0]
    for place, token in enumerate(kept[0, 0]):
        if place // 16 != 1 and token // 16 not in (1, 3):
            assert np.array_equal(rows[page[place // 16], 0, place % 16], before[page[token // 16], 0, token % 16])
    others = np.setdiff1d(np.arange(e.c.pages), page[page >= 0])
    assert np.array_equal(rows[others], before[others])


def test_evictions_recorded(km, gpu):
    rng = np.random.default_rng(10)
    e = Evict(km, rng, 2, 64, 16, [300, 200, 20], 100, 4, 30)
    want = e.check()
    with km.Graph() as g:
        e.call()
    for _ in range(3):
        for again in (g.launch, e.call):
            e.c.blocks.write(e.raw)
            e.w.write(e.weights)
            e.kept.zero()
            km.sync()
            again()
            assert all(np.array_equal(a, b) for a, b in zip(e.results(), want))
    g.destroy()


# ---------------------------------------------------------------- together -----------------------

@pytest.mark.parametrize("kind", [F16, BF16])
def test_a_prompt_from_its_rows_to_a_smaller_cache(km, gpu, kind):
    """As a program uses them: rows are rotated, the prompt attends to itself, its rows go to the cache, a few more tokens are decoded behind the prefix that two answers share, the
    weights of the prompt's tokens are added up, the prompt is cut down to its budget, and decoding goes on from what is left."""
    from test_gpu_rotary import rotated
    from test_gpu_prompt import Prompts
    rng = np.random.default_rng(11)
    heads, group, dim, page, n = 2, 4, 64, 16, 200
    p = Prompts(km, rng, heads, group, dim, [n], [n], kind)
    turns = km.rotary_turns(dim)
    pos, turn_buf = device(km, np.arange(n, dtype=np.int32)), device(km, turns)
    q, k, v = (device(km, to_bits(x, kind)) for x in (p.q, p.k, p.v))
    km.rotary(kind, [km.RotaryRows(q, heads * group), km.RotaryRows(k, heads)], n, dim, turn_buf, pos)
    km.sync()
    from test_gpu_cache4 import from_bits
    read = lambda b, shape: from_bits(b.read(np.uint16, int(np.prod(shape))).view(np.uint16 if kind == BF16 else np.float16), kind).reshape(shape)  # noqa: E731
    for b, x in ((q, p.q.reshape(n, heads * group, dim)), (k, p.k)):
        want, off = rotated(x, np.arange(n), turns, dim, True, False, 1.0)
        assert np.all(np.abs(read(b, x.shape) - want) <= off * 1.01 + {F16: 2.0 ** -11, BF16: 2.0 ** -8}[kind] * np.abs(want) + 2.0 ** -25)
    p.q, p.k = read(q, p.q.shape), read(k, p.k.shape)
    p.check()

    c = Cache(km, rng, heads, dim, page, 20)
    c.write(kind, p.k, p.v, np.arange(n))
    prompt = Queries(km, rng, c, [n], [32], group, kind)  # its last queries look at it again, as cached
    prompt.table = np.arange(prompt.table.shape[1], dtype=np.int32)[None]
    prompt.batch = km.Cache4Batch(1, heads * group, 32, 32, n, device(km, prompt.starts), device(km, np.int32([n])), device(km, prompt.table), prompt.table.shape[1])
    prompt.q = p.q[-32:]
    _, lse = prompt.check()
    weights = weigh(prompt, np.zeros((c.pages, heads, page), np.float32), lse=lse).astype(np.float32)
    want, off = weighed(prompt, np.zeros((c.pages, heads, page), np.float32), lse)
    assert np.all(np.abs(weights - want) <= off)

    # two answers behind the prompt, a page each
    answers = np.array([14, 15])
    more, more_v = ordinary(rng, 6, heads, dim)
    c.write(kind, more, more_v, (answers[:, None] * page + np.arange(3)).reshape(-1))
    hq = heads * group
    from test_gpu_cache4_shared import Shared
    s = Shared.__new__(Shared)
    s.km, s.c, s.kind, s.scale, s.group, s.tokens, s.lengths, s.counts, s.starts = km, c, kind, 0.125, group, 2, [3, 3], [1, 1], np.int32([0, 1, 2])
    s.q = from_bits(to_bits(rng.normal(size=(2, heads, group, dim)), kind), kind)
    s.slots = [(n, np.concatenate([np.arange(n), a * page + np.arange(3)])) for a in answers]
    s.prefix = km.Cache4Batch(1, hq, 2, 2, n, device(km, np.int32([0, 2])), device(km, np.int32([n])), device(km, prompt.table), prompt.table.shape[1])
    s.batch = km.Cache4Batch(2, hq, 2, 1, page, device(km, s.starts), device(km, np.int32([3, 3])), device(km, np.int32(answers[:, None])), 1)
    _, lse = s.check()
    front = Queries(km, rng, c, [n], [2], group, kind)
    front.table, front.q, front.batch = prompt.table, s.q, s.prefix
    before = weights.copy()
    weights = weigh(front, weights, causal=False, lse=lse).astype(np.float32)
    want, off = weighed(front, before, lse, causal=False)
    assert np.all(np.abs(weights - want) <= off)

    # the prompt down to 80 tokens of each head, and the answers from what is left
    keep, first, recent = 80, 4, 16
    w, kept, left = device(km, weights), device(km, np.zeros(heads * keep, np.int32)), device(km, np.zeros(1, np.int32))
    c.dev.evict(s.prefix, w, keep, first, recent, kept, left)
    km.sync()
    kept = kept.read(np.int32, heads * keep).reshape(heads, keep)
    assert left.read(np.int32, 1)[0] == keep
    for h in range(heads):
        at = np.arange(n)
        assert kept[h].tolist() == choice(weights[at // page, h, at % page], n, keep, first, recent)
    old = c.k.copy(), c.v.copy()
    for h in range(heads):
        c.k[:keep, h], c.v[:keep, h] = old[0][kept[h], h], old[1][kept[h], h]
    s.slots = [(keep, np.concatenate([np.arange(keep), a * page + np.arange(3)])) for a in answers]
    s.prefix = km.Cache4Batch(1, hq, 2, 2, n, device(km, np.int32([0, 2])), left, device(km, prompt.table), prompt.table.shape[1])
    s.check()
