"""Attention over prompts on the GPU (csrc/prompt_attend_impl.h) against its definition in 64 bits, within bounds that follow from the types (-m gpu)."""
import numpy as np
import pytest

from test_gpu_cache4 import BF16, F16, UNIT, device, from_bits, to_bits
from test_zz_no_alloc import device_memory_in_use

pytestmark = pytest.mark.gpu


class Prompts:
    def __init__(self, km, rng, heads, group, dim, counts, lengths, kind, loud=1.0, extra=(0, 0), most=(0, 0)):
        """counts, lengths: queries and tokens of each sequence; extra: rows behind the last one's."""
        self.km, self.heads, self.group, self.dim, self.kind, self.counts, self.lengths = km, heads, group, dim, kind, counts, lengths
        self.query_starts, self.token_starts = (np.concatenate([[0], np.cumsum(n)]).astype(np.int32) for n in (counts, lengths))
        self.queries, self.tokens = int(self.query_starts[-1]) + extra[0], int(self.token_starts[-1]) + extra[1]
        rows = lambda *shape: from_bits(to_bits(rng.normal(size=shape), kind), kind)  # noqa: E731
        self.q = from_bits(to_bits(rng.normal(size=(self.queries, heads, group, dim)) * loud, kind), kind)
        self.k, self.v = rows(self.tokens, heads, dim), rows(self.tokens, heads, dim)
        self.scale = 1 / np.sqrt(dim)
        self.most = max(max(counts), most[0]), max(max(lengths), most[1])

    def expected(self, causal=True, scale=None):
        """(out, lse, how far each may be off): a probability has the bits of its type, which half precision has down to 2^-21 of the largest and a part in 2^32 of that below;
        scores and sums have 24 bits with as many terms as they have; the result is rounded to its type."""
        scale = self.scale if scale is None else scale
        shape = (self.queries, self.heads, self.group)
        out, lse = np.zeros(shape + (self.dim,)), np.full(shape, -np.inf)
        off, lse_off = np.zeros_like(out), np.zeros(shape)
        for s, (nq, n) in enumerate(zip(self.counts, self.lengths)):
            rows, at = slice(self.query_starts[s], self.query_starts[s] + nq), slice(self.token_starts[s], self.token_starts[s] + n)
            sees = np.maximum(0, n - nq + 1 + np.arange(nq)) if causal else np.full(nq, n)
            seen = np.arange(n) < sees[:, None]
            some = seen.any(-1)
            for h in range(self.heads):
                k, v = self.k[at, h].astype(np.float64), self.v[at, h].astype(np.float64)
                v_abs = np.where(np.isfinite(v), np.abs(v), 0)
                strange = ~np.isfinite(v)
                for g in range(self.group):
                    if not some.any():
                        continue
                    q = self.q[rows, h, g].astype(np.float64)
                    with np.errstate(invalid="ignore", over="ignore"):
                        score = scale * q @ np.where(np.isfinite(k), k, 0).T
                        bad = ~np.isfinite(k).all(-1)
                        score[:, bad] = np.nan
                        score = np.where(seen, score, -np.inf)
                        top = np.where(some, score.max(-1), 0)[:, None]
                        p = np.where(seen, np.exp(score - top), 0)
                        total = np.maximum(p.sum(-1, keepdims=True), 1e-300)
                        o = p @ np.where(strange, 0, v) / total
                        if strange.any():  # what is no number comes to the rows that see it
                            for t, c in zip(*np.nonzero(strange)):
                                o[seen[:, t], c] += v[t, c]
                        size = p @ v_abs / total
                        length = np.abs(score, where=seen, out=np.zeros_like(score))
                        delta = ((self.dim + 16) * 2.0 ** -23 * (abs(scale) * np.abs(q) @ np.where(np.isfinite(k), np.abs(k), 0).T).max(-1) + 2.0 ** -22 * length.max(-1))[:, None]
                        terms = (sees[:, None] + 64) * 2.0 ** -24
                        out[rows, h, g] = np.where(some[:, None], o, 0)
                        lse[rows, h, g] = np.where(some, top[:, 0] + np.log(total[:, 0]), -np.inf)
                        off[rows, h, g] = UNIT[self.kind] * np.abs(o) + (UNIT[self.kind] + 2 * delta + 2 * terms) * size + (2.0 ** -25 + 2.0 ** -32 * n) * v_abs.max(initial=0)
                        lse_off[rows, h, g] = (delta + terms)[:, 0] + 2.0 ** -21 * (1 + np.abs(np.where(some, lse[rows, h, g], 0)))
        return out, lse, off, lse_off

    def attend(self, causal=True, scale=None, gaps=(0, 0), key_gaps=(0, 0), out_gaps=(0, 0), offset=0, starts=None, fresh=True):
        km, heads, dim = self.km, self.heads * self.group, self.dim
        strides = lambda n, g: (n * (dim + g[0]) + g[1], dim + g[0])  # noqa: E731
        (qt, qh), (kt, kh), (ot, oh) = strides(heads, gaps), strides(self.heads, key_gaps), strides(heads, out_gaps)

        def laid(x, n, t, h):
            flat = np.full(offset + max(1, len(x)) * t, 3, np.float32)
            flat[offset:offset + len(x) * t].reshape(len(x), t)[:, :n * h].reshape(len(x), n, h)[:, :, :dim] = x.reshape(len(x), n, dim)
            return device(km, to_bits(flat, self.kind))

        view = lambda b: km.DeviceView(b.ptr.value + 2 * offset, 0)  # noqa: E731
        self.buffers = laid(self.q, heads, qt, qh), laid(self.k, self.heads, kt, kh), laid(self.v, self.heads, kt, kh)
        out = device(km, np.full(offset + self.queries * ot, 0x5A5A, np.uint16))
        lse = device(km, np.full((self.queries, heads), 77, np.float32))
        starts = (self.query_starts, self.token_starts) if starts is None else starts
        self.prompt = km.Prompt(len(starts[0]) - 1, heads, self.heads, dim, self.queries, self.tokens, *self.most, device(km, starts[0]), device(km, starts[1]))
        q, k, v = (view(b) for b in self.buffers)
        self.call = lambda: self.prompt.attend(self.kind, q, k, v, view(out), self.scale if scale is None else scale, causal=causal, lse=lse, q_token_stride=qt, q_head_stride=qh,  # noqa: E731
                                               token_stride=kt, head_stride=kh, out_token_stride=ot, out_head_stride=oh)
        self.results = out, lse
        self.call()
        km.sync()
        raw = out.read(np.uint16, offset + self.queries * ot)
        rows = raw[offset:].reshape(self.queries, ot)[:, :heads * oh].reshape(self.queries, heads, oh)
        assert (raw[:offset] == 0x5A5A).all() and (rows[:, :, dim:] == 0x5A5A).all(), "written between the rows"
        bits = np.ascontiguousarray(rows[:, :, :dim])
        values = from_bits(bits if self.kind == BF16 else bits.view(np.float16), self.kind)
        self.bits = bits
        return values.reshape(self.queries, self.heads, self.group, dim).astype(np.float64), lse.read(np.float32, self.queries * heads).reshape(self.queries, self.heads, self.group).astype(np.float64)

    def check(self, causal=True, scale=None, **how):
        got, lse = self.attend(causal, scale, **how)
        want, want_lse, off, lse_off = self.expected(causal, scale)
        used = int(self.query_starts[-1])
        assert (self.bits[used:] == 0x5A5A).all() and np.all(lse[used:] == 77), "rows behind the last sequence are left as they were"
        got, lse, want, want_lse, off, lse_off = (x[:used] for x in (got, lse, want, want_lse, off, lse_off))
        empty = np.isneginf(want_lse)
        assert np.array_equal(np.isneginf(lse), empty) and not np.any(got[empty])
        fine = np.isfinite(want)
        assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)])
        far = np.abs(got[fine] - want[fine])
        assert np.all(far <= off[fine]), (far / np.maximum(off[fine], 1e-300)).max()
        some = np.isfinite(want_lse)
        assert np.array_equal(np.isnan(lse), np.isnan(want_lse))
        far = np.abs(lse[some] - want_lse[some])
        assert np.all(far <= lse_off[some]), (far / lse_off[some]).max()
        return got, lse


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,group,dim,lengths", [
    (1, 1, 32, [1]), (2, 4, 64, [1, 31, 32, 33, 64, 63]), (1, 1, 128, [300]), (2, 3, 96, [65, 200]), (1, 8, 128, [127, 2, 90]), (1, 2, 160, [150]), (1, 5, 192, [70, 33]),
    (2, 1, 224, [129]), (1, 2, 256, [260, 31]), (1, 16, 64, [100]), (3, 1, 32, [513])])
def test_whole_prompts(km, gpu, kind, causal, heads, group, dim, lengths):
    rng = np.random.default_rng(dim + group)
    Prompts(km, rng, heads, group, dim, lengths, lengths, kind, extra=(2, 3)).check(causal)


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,group,dim,counts,lengths", [
    (2, 4, 64, [1, 1, 1], [1, 40, 333]), (1, 3, 128, [5, 100, 31], [700, 100, 32]), (1, 1, 96, [1], [1000]), (2, 2, 256, [3, 1], [90, 300]), (1, 7, 32, [64, 1, 20], [65, 500, 21])])
def test_the_last_queries_of_longer_prompts(km, gpu, kind, causal, heads, group, dim, counts, lengths):
    rng = np.random.default_rng(dim + sum(counts))
    Prompts(km, rng, heads, group, dim, counts, lengths, kind).check(causal)


@pytest.mark.parametrize("kind", [F16, BF16])
def test_more_queries_than_tokens_and_empty_sequences(km, gpu, kind):
    """Rows that see nothing: zeros and minus infinity. Sequences without queries, without tokens, without either."""
    rng = np.random.default_rng(2)
    s = Prompts(km, rng, 2, 3, 64, [7, 5, 0, 0, 90], [3, 0, 9, 0, 40], kind, extra=(1, 0))
    got, lse = s.check()
    assert np.isneginf(lse[:4]).all() and np.isneginf(lse[7:12]).all() and np.isfinite(lse[4]).all()
    s.check(causal=False)
    Prompts(km, rng, 1, 2, 32, [4, 3], [0, 0], kind).check()


def test_long_rows(km, gpu):
    """A few queries over many tokens, and one sequence much longer than the others."""
    rng = np.random.default_rng(3)
    for counts, lengths in (([2], [20000]), ([40, 1, 3], [5000, 9, 700])):
        s = Prompts(km, rng, 1, 2, 64, counts, lengths, BF16)
        first = s.check()
        for _ in range(2):
            again = s.attend()
            assert np.array_equal(first[0], again[0]) and np.array_equal(first[1], again[1])


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 96, 256])
def test_strides_and_odd_addresses(km, gpu, kind, dim):
    rng = np.random.default_rng(4)
    s = Prompts(km, rng, 2, 3, dim, [50, 41], [70, 41], kind)
    straight = s.check()
    for how in (dict(gaps=(8, 32), key_gaps=(0, 8), out_gaps=(16, 8), offset=8), dict(gaps=(1, 2), key_gaps=(3, 0), out_gaps=(3, 1), offset=1), dict(key_gaps=(2, 2)), dict(out_gaps=(1, 0))):
        other = s.check(**how)
        assert np.array_equal(straight[0], other[0]) and np.array_equal(straight[1], other[1])


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("scale", [0.0, -0.3, 1e-6, 3.0])
def test_scales(km, gpu, kind, scale):
    rng = np.random.default_rng(5)
    Prompts(km, rng, 1, 2, 64, [90], [120], kind, loud=0.5).check(scale=scale)


@pytest.mark.parametrize("kind,loud", [(BF16, 1e30), (BF16, 1e-30), (F16, 1e-4), (F16, 1e4)])
def test_large_and_small_queries(km, gpu, kind, loud):
    rng = np.random.default_rng(6)
    Prompts(km, rng, 1, 2, 64, [60], [150], kind, loud=loud).check(scale=0.2 / loud)


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("order", ["rising", "falling", "one"])
def test_scores_that_rise_along_the_row(km, gpu, kind, order):
    """The reference of a row is raised many times, never, or once by far; scores of some thousands."""
    rng = np.random.default_rng(7)
    s = Prompts(km, rng, 1, 2, 32, [300], [300], kind)
    ramp = {"rising": np.linspace(-1, 1, 300), "falling": np.linspace(1, -1, 300), "one": np.where(np.arange(300) == 200, 1.0, -1.0)}[order]
    for size in (4.0, 300.0):
        s.q = from_bits(to_bits(np.abs(s.q) + 0.5, kind), kind)
        s.k = from_bits(to_bits(np.repeat(ramp[:, None, None], 32, -1) * size + 0.01 * rng.normal(size=s.k.shape), kind), kind)
        s.check()
        s.check(causal=False)


def test_many_tokens_below_one_that_stands_out(km, gpu):
    """Half precision: 2000 tokens 2^-18 of the largest, which together are as much as 2^-7 of it."""
    rng = np.random.default_rng(8)
    s = Prompts(km, rng, 1, 1, 32, [33], [2000], F16)
    s.q[:] = 1
    s.k[:] = 0
    s.k[500] = 1
    s.v[:] = np.abs(s.v)
    s.v[500] = 0
    s.check(causal=False, scale=18 * np.log(2) / 32)


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("what", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("where", [(39, 5), (100, 0), (129, 31), (70, 17)])
def test_values_that_are_no_numbers(km, gpu, kind, what, where):
    """They come to the rows that see them, and to no other: not to queries before them, nor to other sequences."""
    rng = np.random.default_rng(9)
    s = Prompts(km, rng, 2, 2, 64, [40, 90], [40, 90], kind)
    s.v[where[0], 1, where[1]] = what
    got, _ = s.check()
    assert np.isfinite(got[:, 0]).all() and (~np.isfinite(got[:, 1])).any()
    s.check(causal=False)


@pytest.mark.parametrize("kind", [F16, BF16])
def test_keys_and_queries_that_are_no_numbers(km, gpu, kind):
    rng = np.random.default_rng(10)
    s = Prompts(km, rng, 1, 2, 64, [40, 90], [40, 90], kind)
    s.k[70, 0, 3] = np.nan
    got, lse = s.check()
    assert np.isfinite(got[:70]).all() and np.isnan(got[70:]).all()
    s = Prompts(km, rng, 1, 2, 64, [80], [80], kind)
    s.q[33, 0, 1, 5] = np.nan
    got, lse = s.attend()
    bad = np.zeros((80, 1, 2), bool)
    bad[33, 0, 1] = True
    assert np.array_equal(np.isnan(lse), bad) and np.array_equal(np.isnan(got).all(-1), bad) and np.isfinite(got[~bad]).all()


def test_starts_that_say_nothing(km, gpu):
    """Sequences whose starts are not within the rows have none, bounds may be as loose as they like, and what passes them is cut off."""
    rng = np.random.default_rng(11)
    s = Prompts(km, rng, 1, 2, 64, [30, 40], [30, 40], BF16, most=(70000, 1 << 30))
    want = s.check()
    for starts in (([0, 30, 71], [0, 30, 70]), ([0, 30, -1], [0, 30, 70])):  # the second one's queries
        got, lse = s.attend(starts=tuple(np.int32(x) for x in starts))
        assert np.array_equal(got[:30], want[0][:30]) and (s.bits[30:] == 0x5A5A).all() and np.all(lse[30:] == 77)
    for starts in (([0, 30, 70], [0, 30, 71]), ([0, 30, 70], [0, 30, 20]), ([0, 30, 70], [0, 30, -5])):  # its tokens
        got, lse = s.attend(starts=tuple(np.int32(x) for x in starts))
        assert np.array_equal(got[:30], want[0][:30]) and not got[30:].any() and np.isneginf(lse[30:]).all()
    got, lse = s.attend(starts=(np.int32([-3, 30, 70]), np.int32([0, 30, 70])))
    assert (s.bits[:30] == 0x5A5A).all() and np.array_equal(got[30:], want[0][30:])


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,group,dim,counts,lengths", [
    (2, 4, 128, [1, 3, 1, 0, 2], [3000, 33, 0, 500, 2999]), (1, 1, 32, [200], [2100]), (1, 3, 192, [2, 100], [1500, 40]), (1, 1, 160, [300], [1025]), (1, 2, 256, [5], [2000]),
    (2, 1, 96, [31, 1], [1999, 2000]), (1, 8, 64, [40], [4097]), (1, 1, 224, [90, 90], [64, 1600])])
def test_tokens_in_parts(km, gpu, kind, causal, heads, group, dim, counts, lengths):
    """Few rows over many tokens: work-groups share out the tokens, also of sequences much shorter than the longest, whose last parts are empty."""
    rng = np.random.default_rng(dim + len(counts))
    s = Prompts(km, rng, heads, group, dim, counts, lengths, kind, extra=(1, 0))
    first = s.check(causal)
    again = s.attend(causal, gaps=(1, 0), key_gaps=(0, 1), out_gaps=(1, 1), offset=1)
    assert np.array_equal(first[0], again[0][:len(first[0])]) and np.array_equal(first[1], again[1][:len(first[1])])


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("where", [(0, 0), (1023, 63), (1900, 7), (1999, 40)])
def test_parts_with_values_that_are_no_numbers(km, gpu, kind, where):
    rng = np.random.default_rng(13)
    s = Prompts(km, rng, 2, 2, 64, [120], [2000], kind)
    for what in (np.inf, np.nan):
        s.v[where[0], 1, where[1]] = what
        got, _ = s.check()
        assert np.isfinite(got[:, 0]).all() and (~np.isfinite(got[:, 1])).any()
    s.k[500, 0] = np.nan
    got, lse = s.check()
    assert np.isnan(got[:, 0]).all() and np.isnan(lse[:, 0]).all()


def test_parts_below_one_that_stands_out(km, gpu):
    """Parts whose references are far apart, also further than 32 bits reach."""
    rng = np.random.default_rng(14)
    for far in (10.0, 300.0):
        s = Prompts(km, rng, 1, 1, 32, [3], [3000], BF16)
        s.q[:] = 1
        s.k[:] = from_bits(to_bits(0.01 * rng.normal(size=s.k.shape), BF16), BF16)
        s.k[700] = far / 32
        s.check(causal=False, scale=1.0)


def test_reserved_recorded_and_replayed(km, gpu):
    """Nothing is allocated after kmx_prompt_reserve; recordings outlive the work space."""
    rng = np.random.default_rng(15)
    shapes = [Prompts(km, rng, 2, 4, 128, [1, 2], [3000, 100], BF16), Prompts(km, rng, 1, 4, 128, [60], [2500], F16)]
    want = [(s.attend(), s.results[0].read(np.uint16, s.results[0].nbytes // 2)) for s in shapes]
    shapes[0].results[0].zero()  # (all code is on the device)
    km.check(km.hip_lib().kmx_shutdown())
    km.Prompt.reserve(128)
    km.sync()
    before = device_memory_in_use()

    def same(s, bits):
        km.sync()
        return np.array_equal(s.results[0].read(np.uint16, s.results[0].nbytes // 2), bits)

    for s, (_, bits) in zip(shapes, want):
        s.results[0].write(np.zeros(s.results[0].nbytes, np.uint8))
        s.call()
        assert same(s, bits)
    assert device_memory_in_use() == before
    graphs = []
    for s in shapes:
        with km.Graph() as g:
            s.call()
        graphs.append(g)
    km.check(km.hip_lib().kmx_shutdown())
    for _ in range(3):
        for s, g, (_, bits) in zip(shapes, graphs, want):
            s.results[0].write(np.zeros(s.results[0].nbytes, np.uint8))
            g.launch()
            assert same(s, bits)
            s.call()
    for g in graphs:
        g.destroy()


def test_recorded_and_on_a_stream_of_the_callers(km, gpu):
    import ctypes
    rng = np.random.default_rng(12)
    s = Prompts(km, rng, 2, 2, 64, [100, 3], [100, 3000], BF16)
    s.check()
    out, lse = s.results
    want = out.read(np.uint16, out.nbytes // 2), lse.read(np.float32, lse.nbytes // 4)

    def same():
        km.sync()
        ok = np.array_equal(out.read(np.uint16, out.nbytes // 2), want[0]) and np.array_equal(lse.read(np.float32, lse.nbytes // 4), want[1])
        out.write(np.zeros(out.nbytes, np.uint8))
        lse.write(np.zeros(lse.nbytes, np.uint8))
        return ok

    with km.Graph() as g:
        s.call()
    for _ in range(3):
        out.write(np.zeros(out.nbytes, np.uint8))
        g.launch()
        assert same()
        s.call()
        assert same()
    g.destroy()
    hip = ctypes.CDLL(next(line.split()[-1] for line in open("/proc/self/maps") if "libamdhip64" in line))  # the runtime that the library runs on
    stream = ctypes.c_void_p()
    assert hip.hipStreamCreateWithFlags(ctypes.byref(stream), 1) == 0  # waits for no other stream
    km.check(km.hip_lib().kmx_set_stream(stream))
    try:
        for _ in range(3):
            s.call()
            assert same()
    finally:
        km.sync()
        km.check(km.hip_lib().kmx_set_stream(None))
        assert hip.hipStreamDestroy(stream) == 0
