"""Attention to prefixes that sequences share (kmx_cache4_attend_shared) against one softmax over prefix and own tokens in 64 bits (-m gpu)."""
import numpy as np
import pytest

from test_gpu_cache4 import BF16, F16, Cache, Queries, device, from_bits, to_bits
from test_zz_no_alloc import device_memory_in_use

pytestmark = pytest.mark.gpu


class Shared:
    """Prefixes of some lengths, the first `members[p]` sequences of each in order; sequences behind the last member have no prefix."""

    def __init__(self, km, rng, heads, group, dim, page, prefixes, members, lengths, counts, kind, loud=1.0, most=None):
        self.km, self.prefixes, self.members = km, prefixes, members
        pages = sum(-(-n // page) for n in list(prefixes) + list(lengths))
        self.c = Cache(km, rng, heads, dim, page, pages + 2)
        both = Queries(km, rng, self.c, list(prefixes) + list(lengths), [0] * len(prefixes) + list(counts), group, kind, loud=loud).fill(rng)
        self.q, self.kind, self.scale, self.group, self.tokens, self.lengths, self.counts = both.q, kind, both.scale, group, both.tokens, lengths, counts
        self.front, self.table = both.table[:len(prefixes)], both.table[len(prefixes):]
        self.starts = both.starts[len(prefixes):]
        ends = np.cumsum([0] + list(members))
        self.prefix_starts = self.starts[ends]
        hq, width, longest = heads * group, both.table.shape[1], most or max(list(prefixes) + list(lengths) + [1])
        rows = max(1, int(np.diff(self.prefix_starts).max(initial=1)))
        table = lambda t: device(km, np.ascontiguousarray(t))  # noqa: E731
        self.prefix = km.Cache4Batch(len(prefixes), hq, self.tokens, rows, longest, device(km, self.prefix_starts), device(km, np.int32(prefixes)), table(self.front), width)
        self.batch = km.Cache4Batch(len(lengths), hq, self.tokens, max(counts), longest, device(km, self.starts), device(km, np.int32(lengths)), table(self.table), width)
        # one sequence of each: the prefix's tokens and then its own (whole pages apart, so a list of places and not a table)
        self.slots = []
        for s, n in enumerate(lengths):
            p = int(np.searchsorted(ends, s, side="right")) - 1
            ahead = prefixes[p] if p < len(prefixes) else 0
            at, own = np.arange(ahead), np.arange(n)
            self.slots.append((ahead, np.concatenate([self.front[min(p, len(prefixes) - 1), at // page] * page + at % page if ahead else at, self.table[s, own // page] * page + own % page]).astype(int)))

    def expected(self, causal=True, scale=None):
        """As Queries.expected, over the tokens of both; the probabilities of each part are rounded against the largest of that part, so no further off than together."""
        c, scale, unit = self.c, self.scale if scale is None else scale, {F16: 2.0 ** -11, BF16: 2.0 ** -8}[self.kind]
        shape = (self.tokens, c.heads, self.group)
        out, lse = np.zeros(shape + (c.dim,)), np.full(shape, -np.inf)
        off, lse_off = np.zeros_like(out), np.zeros(shape)
        for s, (ahead, slots) in enumerate(self.slots):
            for i in range(self.counts[s]):
                own = max(0, self.lengths[s] - self.counts[s] + i + 1) if causal else self.lengths[s]
                use = slots[:ahead + own]
                if not len(use):
                    continue
                for h in range(c.heads):
                    t = self.starts[s] + i
                    k, v, q = c.k[use, h].astype(np.float64), c.v[use, h].astype(np.float64), self.q[t, h].astype(np.float64)
                    score = scale * q @ k.T
                    top = score.max(-1, keepdims=True)
                    p = np.exp(score - top)
                    total = p.sum(-1, keepdims=True)
                    out[t, h], lse[t, h] = p @ v / total, top[:, 0] + np.log(total[:, 0])
                    delta = ((c.dim + 16) * 2.0 ** -23 * (abs(scale) * np.abs(q) @ np.abs(k).T).max(-1) + 2.0 ** -22 * np.abs(score).max(-1))[:, None]
                    terms = (len(use) + 128) * 2.0 ** -24
                    off[t, h] = unit * np.abs(out[t, h]) + (2.0 ** -11 + 2 * delta + 2 * terms) * (p @ np.abs(v) / total) + 2.0 ** -25 * np.abs(v).max()
                    lse_off[t, h] = delta[:, 0] + terms + 2.0 ** -21 * (1 + np.abs(lse[t, h]))
        return out, lse, off, lse_off

    def attend(self, causal=True, scale=None, gaps=(0, 0), out_gaps=(0, 0), offset=0, prefix=None, batch=None):
        km, c = self.km, self.c
        heads = c.heads * self.group
        strides = lambda g: ((c.dim + g[0]) * heads + g[1], c.dim + g[0])  # noqa: E731
        (qt, qh), (ot, oh) = strides(gaps), strides(out_gaps)
        flat = np.full((self.tokens, qt), 3, np.float32)
        flat[:, :heads * qh].reshape(self.tokens, heads, qh)[:, :, :c.dim] = self.q.reshape(self.tokens, heads, c.dim)
        q = device(km, to_bits(np.concatenate([np.zeros(offset, np.float32), flat.reshape(-1)]), self.kind))
        out = device(km, np.full(offset + self.tokens * ot, 0x5A5A, np.uint16))
        lse = device(km, np.full((self.tokens, heads), 77, np.float32))
        view = lambda b: km.DeviceView(b.ptr.value + 2 * offset, 0)  # noqa: E731
        self.buffers = q, out, lse
        self.call = lambda: c.dev.attend_shared(prefix or self.prefix, batch or self.batch, self.kind, view(q), view(out), self.scale if scale is None else scale, causal=causal, lse=lse,  # noqa: E731
                                                q_token_stride=qt, q_head_stride=qh, out_token_stride=ot, out_head_stride=oh)
        self.call()
        return self.results(ot, oh, offset)

    def results(self, ot=None, oh=None, offset=0):
        c, heads = self.c, self.c.heads * self.group
        oh = c.dim if oh is None else oh
        ot = heads * oh if ot is None else ot
        self.km.sync()
        raw = self.buffers[1].read(np.uint16, offset + self.tokens * ot)
        rows = raw[offset:].reshape(self.tokens, ot)[:, :heads * oh].reshape(self.tokens, heads, oh)
        assert (raw[:offset] == 0x5A5A).all() and (rows[:, :, c.dim:] == 0x5A5A).all(), "written between the rows"
        self.bits = np.ascontiguousarray(rows[:, :, :c.dim])
        values = from_bits(self.bits if self.kind == BF16 else self.bits.view(np.float16), self.kind)
        return values.reshape(self.tokens, c.heads, self.group, c.dim).astype(np.float64), self.buffers[2].read(np.float32, self.tokens * heads).reshape(self.tokens, c.heads, self.group).astype(np.float64)

    def check(self, causal=True, scale=None, **how):
        got, lse = self.attend(causal, scale, **how)
        want, want_lse, off, lse_off = self.expected(causal, scale)
        empty = np.isneginf(want_lse)
        assert np.array_equal(np.isneginf(lse), empty) and not np.any(got[empty])
        assert np.all(np.abs(got - want) <= off), (np.abs(got - want) / np.maximum(off, 1e-300)).max()
        far = np.abs(lse[~empty] - want_lse[~empty])
        assert np.all(far <= lse_off[~empty]), (far / lse_off[~empty]).max()
        return got, lse


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("heads,group,dim,page,prefixes,members,lengths,counts", [
    (1, 1, 32, 16, [1], [1], [1], [1]), (2, 4, 64, 32, [40, 64], [3, 2], [5, 1, 33, 64, 2], [1] * 5), (2, 3, 96, 64, [100, 0, 17], [1, 2, 1], [3, 70, 9, 1], [1] * 4),
    (1, 8, 128, 64, [300], [20], [1 + 3 * n for n in range(20)], [1] * 20),                       # more than 64 rows of a head look at the prefix
    (2, 5, 160, 16, [130], [2], [20, 41], [4, 7]), (1, 16, 192, 128, [500, 3], [4, 1], [9, 1, 130, 64, 2], [1, 1, 2, 1, 2]),
    (1, 2, 224, 64, [90], [3], [30, 2, 5], [1, 2, 5]), (2, 2, 256, 16, [77, 200], [2, 3], [4, 8, 15, 16, 23], [1, 3, 1, 2, 1]),
    (1, 4, 64, 64, [200], [2], [100, 90], [90, 40])])                                              # and at their own tokens
@pytest.mark.parametrize("causal", [True, False])
def test_prefixes_and_own_tokens(km, gpu, kind, heads, group, dim, page, prefixes, members, lengths, counts, causal):
    rng = np.random.default_rng(dim + len(lengths))
    Shared(km, rng, heads, group, dim, page, prefixes, members, lengths, counts, kind).check(causal)


@pytest.mark.parametrize("counts", [[1] * 6, [30] * 6])
def test_long_prefixes_in_parts(km, gpu, counts):
    rng = np.random.default_rng(1)
    s = Shared(km, rng, 1, 4, 64, 64, [9000, 3100], [4, 2], [40, 300, 2000, 31, 700, 60], counts, BF16)
    first = s.check()
    for _ in range(3):
        again = s.attend()
        assert np.array_equal(first[0], again[0]) and np.array_equal(first[1], again[1])


@pytest.mark.parametrize("group,counts", [(2, 1), (2, 50)])
def test_sequences_without_a_prefix_and_prefixes_without_sequences(km, gpu, group, counts):
    """Rows that no prefix has see their own tokens only; of a prefix of no tokens nothing; own sequences may be empty too."""
    rng = np.random.default_rng(2)
    Shared(km, rng, 2, group, 64, 16, [50, 30], [2, 0], [60, 55, 51, 70], [counts] * 4, F16).check()
    Shared(km, rng, 2, group, 64, 16, [0, 30], [2, 1], [60, 0, 0, 0], [counts] * 4, F16).check()
    s = Shared(km, rng, 1, group, 64, 16, [50], [2], [9, 4], [1, 1], F16)
    none = km.Cache4Batch(0, group, s.tokens, 1, 50, device(km, s.starts), device(km, s.starts), device(km, s.table), s.table.shape[1])
    got, lse = s.attend(prefix=none)
    q, out, own = s.buffers[0], device(km, np.zeros(2 * group * 64, np.uint16)), device(km, np.zeros(2 * group, np.float32))
    s.c.dev.attend(s.batch, F16, q, out, s.scale, lse=own)
    km.sync()
    assert np.array_equal(out.read(np.uint16, 2 * group * 64), s.bits.reshape(-1)) and np.array_equal(own.read(np.float32, 2 * group), lse.reshape(-1).astype(np.float32))


def test_rows_of_no_sequence_are_left_as_they_were(km, gpu):
    rng = np.random.default_rng(3)
    s = Shared(km, rng, 1, 2, 64, 16, [50], [3], [9, 4, 20], [1, 1, 1], BF16)
    full, _ = s.attend()
    fewer = km.Cache4Batch(2, 2, s.tokens, 1, 50, device(km, s.starts), device(km, np.int32(s.lengths)), device(km, s.table), s.table.shape[1])
    got, lse = s.attend(batch=fewer)
    assert np.array_equal(got[:2], full[:2]) and (s.bits[2] == 0x5A5A).all() and np.all(lse[2] == 77)


def test_starts_of_prefixes_that_say_nothing(km, gpu):
    """Prefixes whose rows are not within the queries have none; rows beyond max_queries see their own tokens only."""
    rng = np.random.default_rng(4)
    s = Shared(km, rng, 1, 2, 64, 16, [50], [3], [9, 4, 20], [1, 1, 1], BF16)
    full, full_lse = s.attend()
    own = Shared.__new__(Shared)
    make = lambda starts, most: km.Cache4Batch(1, 2, s.tokens, most, 50, device(km, np.int32(starts)), device(km, np.int32([50])), device(km, s.front), s.front.shape[1])  # noqa: E731
    alone, alone_lse = s.attend(prefix=make([0, 0], 3))
    assert not np.array_equal(alone, full)
    for starts in ([0, 4], [-1, 3], [3, 2], [1 << 30, (1 << 30) + 2]):
        got, lse = s.attend(prefix=make(starts, 3))
        assert np.array_equal(got, alone) and np.array_equal(lse, alone_lse)
    got, lse = s.attend(prefix=make([0, 3], 2))
    assert np.array_equal(got[:2], full[:2]) and np.array_equal(got[2], alone[2])
    got, lse = s.attend(prefix=make([1, 3], 3))
    assert np.array_equal(got[1:], full[1:]) and np.array_equal(got[0], alone[0]) and np.array_equal(lse[0], alone_lse[0])
    del own


@pytest.mark.parametrize("counts", [1, 40])
def test_strides_and_odd_addresses(km, gpu, counts):
    rng = np.random.default_rng(5)
    s = Shared(km, rng, 2, 3, 96, 32, [200], [2], [50, 45], [counts] * 2, BF16)
    straight = s.check()
    for how in (dict(gaps=(8, 32), out_gaps=(16, 8), offset=8), dict(gaps=(1, 2), out_gaps=(3, 1), offset=1)):
        other = s.check(**how)
        assert np.array_equal(straight[0], other[0]) and np.array_equal(straight[1], other[1])


@pytest.mark.parametrize("scale,loud", [(0.0, 1.0), (-0.3, 0.5), (4.0, 0.5), (0.2e-30, 1e30)])
def test_scales(km, gpu, scale, loud):
    """Where one part's scores are far above the other's, the other adds nothing."""
    rng = np.random.default_rng(6)
    Shared(km, rng, 1, 2, 64, 16, [100], [3], [40, 3, 80], [1, 1, 1], BF16, loud=loud).check(scale=scale)


def test_pages_that_are_not_there(km, gpu):
    rng = np.random.default_rng(7)
    s = Shared(km, rng, 1, 2, 64, 16, [64], [2], [20, 33], [1, 1], BF16)
    want = s.attend()
    front = s.front.copy()
    front[0, 1:4] = [-1, s.c.pages, 1 << 30]
    cut = km.Cache4Batch(1, 2, s.tokens, 2, 64, device(km, s.prefix_starts), device(km, np.int32([64])), device(km, front), front.shape[1])
    got, lse = s.attend(prefix=cut)
    s.slots = [(16, np.concatenate([x[:16], x[64:]])) for _, x in s.slots]
    expected, expected_lse, off, lse_off = s.expected()
    assert np.all(np.abs(got - expected) <= off) and np.all(np.abs(lse - expected_lse) <= lse_off) and not np.array_equal(got, want[0])


def test_reserved_recorded_and_replayed(km, gpu):
    """Nothing is allocated after kmx_cache4_reserve_shared, for smaller batches neither; recordings outlive the work space."""
    rng = np.random.default_rng(8)
    large = Shared(km, rng, 2, 4, 64, 16, [3000], [6], [200, 100, 31, 5, 60, 900], [1] * 6, BF16)
    small = Shared(km, rng, 2, 4, 64, 16, [1700], [3], [20, 10, 31], [1] * 3, BF16)
    want = [(s.attend(), s.bits.copy()) for s in (large, small)]
    large.buffers[1].zero()  # (all code is on the device)
    km.check(km.hip_lib().kmx_shutdown())
    large.c.dev.reserve_shared(large.prefix, large.batch)
    km.sync()
    before = device_memory_in_use()
    for s, (w, bits) in zip((large, small), want):
        s.buffers[1].zero()
        s.call()
        got = s.results()
        assert np.array_equal(got[0], w[0]) and np.array_equal(got[1], w[1])
    assert device_memory_in_use() == before
    graphs = []
    for s in (large, small):
        with km.Graph() as g:
            s.call()
        graphs.append(g)
    km.check(km.hip_lib().kmx_shutdown())
    for _ in range(3):
        for s, g, (w, bits) in zip((large, small), graphs, want):
            s.buffers[1].zero()
            g.launch()
            got = s.results()
            assert np.array_equal(got[0], w[0]) and np.array_equal(got[1], w[1])
            s.call()
    for g in graphs:
        g.destroy()
