"""The 4-bit cache on the GPU (csrc/cache4.hip, cache4_attend_impl.h) against its definition in numpy: quantised rows bit for bit, chosen pages
number for number, attention in 64 bits within bounds that follow from the types (-m gpu)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

F32, F16, BF16 = 0, 1, 2
UNIT = {F16: 2.0 ** -11, BF16: 2.0 ** -8}  # rounding of a result


# ---------------------------------------------------------------- numbers ------------------------

def to_bits(x, kind):
    """float32 values in the type, as stored."""
    x = np.ascontiguousarray(x, dtype=np.float32)
    if kind == F32:
        return x
    if kind == F16:
        return x.astype(np.float16)
    u = x.view(np.uint32)
    rounded = ((u.astype(np.uint64) + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), (u >> 16).astype(np.uint16) | 0x40, rounded)


def from_bits(b, kind):
    if kind == BF16:
        return (b.astype(np.uint32) << 16).view(np.float32)
    return b.astype(np.float32)


def scales_of(x):
    """Scales of groups of 32 (..., 32) float32: the largest magnitude with 5 significant bits, at most 63488, as half precision holds it."""
    largest = np.fmax.reduce(np.abs(x), axis=-1, initial=0).astype(np.float64)  # (NaN left out)
    part, power = np.frexp(np.minimum(largest, 65504.0))
    return np.minimum(np.ldexp(np.round(part * 32) / 32, power), 63488.0).astype(np.float16)


def held(x, levels):
    """What the cache holds of rows (tokens, heads, dim) with levels (heads, 8), in float32, exactly."""
    t, heads, dim = x.shape
    g = np.float32(x).reshape(t, heads, dim // 32, 32)
    scale = scales_of(g).astype(np.float32)[..., None]
    lv = levels.astype(np.float32)
    middle = (lv[:, :-1] + lv[:, 1:]) * np.float32(0.5)
    with np.errstate(invalid="ignore"):
        index = sum((np.abs(g) > scale * middle[None, :, None, None, j]).astype(np.int64) for j in range(7))
        magnitude = scale * np.take_along_axis(np.broadcast_to(lv[None, :, None, :], (t, heads, dim // 32, 8)), index, -1)
        return np.where(g < 0, -magnitude, magnitude).reshape(t, heads, dim).astype(np.float32)


def some_levels(rng, km, heads):
    base = np.array([0.0381, 0.1172, 0.2036, 0.3003, 0.4097, 0.5396, 0.7075, 0.9712])
    return km.cache4_round_levels(np.minimum(base * (1 + 0.04 * (rng.random((heads, 2, 8)) - 0.5)), 1.0))


class Cache:
    """A cache on the device, and beside it what every place holds."""

    def __init__(self, km, rng, heads, dim, page, pages, garbage=0xFF):
        self.km, self.heads, self.dim, self.page, self.pages = km, heads, dim, page, pages
        blocks, bounds = km.Cache4.sizes(heads, dim, page, pages)
        self.blocks, self.bounds = km.DeviceBuffer(max(16, blocks)), km.DeviceBuffer(max(16, bounds))
        self.blocks.write(np.full(blocks, garbage, np.uint8))
        self.bounds.write(np.full(bounds, garbage, np.uint8))
        self.levels_host = some_levels(rng, km, heads)
        self.levels = km.DeviceBuffer(self.levels_host.nbytes)
        self.levels.write(self.levels_host)
        self.dev = km.Cache4(heads, dim, page, pages, self.levels, self.blocks, self.bounds)
        self.k = np.zeros((pages * page, heads, dim), np.float32)
        self.v = np.zeros((pages * page, heads, dim), np.float32)

    def write(self, kind, keys, values, slots, gaps=(0, 0), offset=0):
        """keys, values: float32; stored with `gaps` elements between heads and tokens, from element `offset` on."""
        km, t = self.km, len(slots)
        hs = self.dim + gaps[0]
        ts = self.heads * hs + gaps[1]
        buf = []
        for rows in (keys, values):
            flat = np.full(offset + max(1, t) * ts, 7, np.float32)
            for i in range(t):
                for h in range(self.heads):
                    flat[offset + i * ts + h * hs:][:self.dim] = rows[i, h]
            bits = to_bits(flat, kind)
            b = km.DeviceBuffer(bits.nbytes)
            b.write(bits)
            buf.append((b, bits))
        slot_buf = device(km, np.asarray(slots, np.int32))
        item = buf[0][1].itemsize
        self.dev.write(kind, km.DeviceView(buf[0][0].ptr.value + offset * item, 0), km.DeviceView(buf[1][0].ptr.value + offset * item, 0), slot_buf, t, ts, hs)
        km.sync()
        keep = [i for i, s in enumerate(slots) if 0 <= s < self.pages * self.page]
        if keep:
            at = np.asarray(slots)[keep]
            self.k[at] = held(from_bits(to_bits(keys, kind), kind)[keep], self.levels_host[:, 0])
            self.v[at] = held(from_bits(to_bits(values, kind), kind)[keep], self.levels_host[:, 1])

    def read(self, kind, slots, gaps=(0, 0), offset=0):
        km, t = self.km, len(slots)
        hs = self.dim + gaps[0]
        ts = self.heads * hs + gaps[1]
        item = 4 if kind == F32 else 2
        pattern = np.full((offset + max(1, t) * ts) * item, 0x5A, np.uint8)
        out = [km.DeviceBuffer(pattern.nbytes) for _ in range(2)]
        for b in out:
            b.write(pattern)
        slot_buf = device(km, np.asarray(slots, np.int32))
        self.dev.read(kind, km.DeviceView(out[0].ptr.value + offset * item, 0), km.DeviceView(out[1].ptr.value + offset * item, 0), slot_buf, t, ts, hs)
        km.sync()
        got = []
        for b in out:
            raw = b.read(np.uint8, pattern.nbytes)
            bits = raw.view({F32: np.float32, F16: np.float16, BF16: np.uint16}[kind])[offset:][:t * ts].reshape(t, ts)[:, :self.heads * hs].reshape(t, self.heads, hs)
            rest = raw.reshape(-1, item)[:offset]
            assert (rest == 0x5A).all() and (np.ascontiguousarray(bits[:, :, self.dim:]).view(np.uint8) == 0x5A).all(), "written between the rows"
            got.append(bits[:, :, :self.dim])
        return got


def device(km, array):
    a = np.ascontiguousarray(array)
    b = km.DeviceBuffer(max(16, a.nbytes))
    if a.nbytes:
        b.write(a)
    return b


def same_bits(a, b):
    a, b = np.ascontiguousarray(a), np.ascontiguousarray(b)
    whole = {2: np.uint16, 4: np.uint32}[a.itemsize]
    x, y = a.view(whole), b.view(whole)
    zero = 1 << (8 * a.itemsize - 1)
    return np.array_equal(np.where(x == zero, 0, x), np.where(y == zero, 0, y))  # (one zero)


def ordinary(rng, tokens, heads, dim):
    loud = 1 + 4 * (rng.random((heads, dim)) < 0.05)
    return np.float32(rng.normal(size=(tokens, heads, dim)) * loud), np.float32(rng.normal(size=(tokens, heads, dim)) * (0.2 + rng.random((tokens, heads, 1))))


# ---------------------------------------------------------------- rows ---------------------------

@pytest.mark.parametrize("kind", [F32, F16, BF16])
@pytest.mark.parametrize("heads,dim,page,tokens", [(1, 32, 16, 1), (2, 64, 32, 15), (3, 96, 64, 16), (4, 128, 16, 17), (2, 160, 128, 100), (5, 192, 256, 63), (1, 224, 64, 65), (2, 256, 16, 33)])
@pytest.mark.parametrize("order", ["run", "late run", "scattered"])
def test_rows_are_held_as_defined(km, gpu, kind, heads, dim, page, tokens, order):
    rng = np.random.default_rng(dim * 3 + tokens)
    pages = (tokens + 5) // page + 3
    c = Cache(km, rng, heads, dim, page, pages)
    keys, values = ordinary(rng, tokens, heads, dim)
    start = {"run": page, "late run": 5, "scattered": 0}[order]
    slots = start + np.arange(tokens) if order != "scattered" else rng.permutation(pages * page)[:tokens]
    c.write(kind, keys, values, slots)
    for back in (F32, kind):
        k, v = c.read(back, slots)
        assert same_bits(k, to_bits(c.k[slots], back)) and same_bits(v, to_bits(c.v[slots], back))
    assert np.all(to_bits(c.k[slots], F16).astype(np.float64) == c.k[slots]), "numbers of half precision"


def test_single_tokens_leave_their_neighbours_alone(km, gpu):
    rng = np.random.default_rng(8)
    c = Cache(km, rng, 3, 64, 16, 6, garbage=0)
    keys, values = ordinary(rng, 96, 3, 64)
    order = rng.permutation(96)
    for n in range(0, 96, 7):   # a few at a time, anywhere
        part = order[n:n + 7]
        c.write(BF16, keys[part], values[part], part)
    k, v = c.read(F32, np.arange(96))
    assert same_bits(k, c.k) and same_bits(v, c.v)


@pytest.mark.parametrize("kind", [F32, F16, BF16])
@pytest.mark.parametrize("gaps,offset", [((8, 16), 8), ((1, 3), 5)])
def test_rows_with_gaps_and_odd_addresses(km, gpu, kind, gaps, offset):
    rng = np.random.default_rng(4)
    c = Cache(km, rng, 3, 96, 32, 3)
    keys, values = ordinary(rng, 40, 3, 96)
    slots = rng.permutation(96)[:40]
    c.write(kind, keys, values, slots, gaps, offset)
    k, v = c.read(kind, slots, gaps, offset)
    assert same_bits(k, to_bits(c.k[slots], kind)) and same_bits(v, to_bits(c.v[slots], kind))


def test_places_that_are_not_there(km, gpu):
    rng = np.random.default_rng(5)
    c = Cache(km, rng, 2, 32, 16, 2, garbage=0)
    before = c.blocks.read(np.uint8, c.blocks.nbytes)
    keys, values = ordinary(rng, 6, 2, 32)
    c.write(F32, keys, values, [-1, 32, 1 << 30, -(1 << 31), (1 << 31) - 1, 33])
    assert np.array_equal(before, c.blocks.read(np.uint8, c.blocks.nbytes))
    c.write(F32, keys, values, [3, -1, 40, 5, -7, 31])
    k, v = c.read(F32, [3, -1, 40, 5, -7, 31])
    for got, want in ((k, c.k), (v, c.v)):
        assert same_bits(got[[0, 3, 5]], want[[3, 5, 31]]) and not np.any(got[[1, 2, 4]])


def test_unusual_numbers(km, gpu):
    """Zeros, groups of zeros, numbers at the edge between two levels, below and beyond half precision, infinities and NaN."""
    rng = np.random.default_rng(6)
    c = Cache(km, rng, 1, 64, 16, 2, garbage=0)
    lv = c.levels_host[0].astype(np.float32)
    x = np.float32(rng.normal(size=(12, 1, 64)))
    x[0] = 0
    x[1, 0, :32] = 0
    x[2, 0, :9] = [-0.0, 0.0, 1e-30, -1e-30, 1e-45, np.nan, -np.nan, 3, -3]
    x[3, 0, 5], x[3, 0, 40] = np.inf, -np.inf
    x[4] = np.nan
    x[5, 0, 0], x[5, 0, 33] = 3e38, 65504
    x[6] *= 1e-6
    x[7] *= 1e-9
    for row, which in ((8, 0), (9, 1)):  # a scale of 1, and the very edges, one place below and one above
        edge = (lv[which][:-1] + lv[which][1:]) * np.float32(0.5)
        x[row] = 0
        x[row, 0, 0] = 1
        x[row, 0, 1:8], x[row, 0, 8:15], x[row, 0, 15:22] = edge, np.nextafter(edge, 0), -np.nextafter(edge, np.float32(2))
    x[10, 0, 0] = 1.03125 * 2  # halfway between 5 bits: to the even one
    x[11, 0, :32] = np.ldexp(1.0, rng.integers(-20, 5, 32))
    c.write(F32, x, x, np.arange(12))
    k, v = c.read(F32, np.arange(12))
    assert same_bits(k, c.k[:12]) and same_bits(v, c.v[:12])
    assert np.isfinite(k).all() and not np.any(k[0]) and np.abs(k[3, 0, 5]) <= 63488


# ---------------------------------------------------------------- attention ----------------------

class Queries:
    """Sequences of given lengths with pages of a cache, and queries of their last tokens."""

    def __init__(self, km, rng, cache, lengths, counts, group, kind, extra=1, loud=1.0):
        self.km, self.c, self.lengths, self.counts, self.group, self.kind = km, cache, lengths, counts, group, kind
        page = cache.page
        used = [-(-n // page) for n in lengths]
        width = max(1, max(used)) + extra
        where = rng.permutation(cache.pages)
        assert sum(used) <= cache.pages
        self.table = np.full((len(lengths), width), -1, np.int32)
        at = 0
        for s, n in enumerate(used):
            self.table[s, :n] = where[at:at + n]
            at += n
        self.starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        self.tokens = int(self.starts[-1])
        self.q = from_bits(to_bits(rng.normal(size=(self.tokens, cache.heads, group, cache.dim)) * loud, kind), kind)
        self.scale = 1 / np.sqrt(cache.dim)
        self.batch = km.Cache4Batch(len(lengths), cache.heads * group, self.tokens, max(counts), max(lengths), device(km, self.starts), device(km, np.int32(lengths)),
                                    device(km, self.table), width)

    def fill(self, rng, kind=F32):
        """Rows for all tokens of all sequences."""
        for s, n in enumerate(self.lengths):
            if n:
                at = np.arange(n)
                self.c.write(kind, *ordinary(rng, n, self.c.heads, self.c.dim), self.table[s, at // self.c.page] * self.c.page + at % self.c.page)
        return self

    def sees(self, s, i, causal=True):
        return max(0, self.lengths[s] - self.counts[s] + i + 1) if causal else self.lengths[s]

    def expected(self, causal=True, chosen=None, scale=None):
        """(out, lse, how far each may be off): the definition in 64 bits, and bounds from the roundings that the kernels make: a probability to 11 bits,
        scores and sums in 24 with as many terms as they have, the result to its type."""
        c, scale = self.c, self.scale if scale is None else scale
        shape = (self.tokens, c.heads, self.group)
        out, lse = np.zeros(shape + (c.dim,)), np.full(shape, -np.inf)
        off, lse_off = np.zeros_like(out), np.zeros(shape)
        for s, n in enumerate(self.lengths):
            at = np.arange(n)
            pages = self.table[s, at // c.page]
            there = (pages >= 0) & (pages < c.pages)
            slots = np.where(there, pages, 0) * c.page + at % c.page
            for i in range(self.counts[s]):
                t = self.starts[s] + i
                for h in range(c.heads):
                    mask = there & (at < self.sees(s, i, causal))
                    if chosen is not None:
                        mask &= np.isin(at // c.page, chosen[t, h])
                    if not mask.any():
                        continue
                    k, v = c.k[slots[mask], h].astype(np.float64), c.v[slots[mask], h].astype(np.float64)
                    q = self.q[t, h].astype(np.float64)
                    score = scale * q @ k.T
                    top = score.max(-1, keepdims=True)
                    p = np.exp(score - top)
                    total = p.sum(-1, keepdims=True)
                    out[t, h] = p @ v / total
                    lse[t, h] = top[:, 0] + np.log(total[:, 0])
                    delta = ((c.dim + 16) * 2.0 ** -23 * (abs(scale) * np.abs(q) @ np.abs(k).T).max(-1) + 2.0 ** -22 * np.abs(score).max(-1))[:, None]
                    terms = (mask.sum() + 64) * 2.0 ** -24
                    off[t, h] = UNIT[self.kind] * np.abs(out[t, h]) + (2.0 ** -11 + 2 * delta + 2 * terms) * (p @ np.abs(v) / total) + 2.0 ** -25 * np.abs(v).max()
                    lse_off[t, h] = delta[:, 0] + terms + 2.0 ** -21 * (1 + np.abs(lse[t, h]))
        return out, lse, off, lse_off

    def attend(self, causal=True, chosen=None, scale=None, gaps=(0, 0), out_gaps=(0, 0), offset=0):
        km, c = self.km, self.c
        heads = c.heads * self.group
        strides = lambda g: ((c.dim + g[0]) * heads + g[1], c.dim + g[0])  # noqa: E731
        (qt, qh), (ot, oh) = strides(gaps), strides(out_gaps)
        flat = np.full(offset + self.tokens * qt, 3, np.float32)
        for t in range(self.tokens):
            flat[offset + t * qt:][:heads * qh].reshape(heads, qh)[:, :c.dim] = self.q[t].reshape(heads, c.dim)
        q = device(km, to_bits(flat, self.kind))
        out = device(km, np.full(offset + self.tokens * ot, 0x5A5A, np.uint16))
        lse = device(km, np.full((self.tokens, heads), 77, np.float32))
        listed = {} if chosen is None else dict(chosen=device(km, np.int32(chosen)), top=chosen.shape[2])
        c.dev.attend(self.batch, self.kind, km.DeviceView(q.ptr.value + 2 * offset, 0), km.DeviceView(out.ptr.value + 2 * offset, 0), self.scale if scale is None else scale,
                     causal=causal, lse=lse, q_token_stride=qt, q_head_stride=qh, out_token_stride=ot, out_head_stride=oh, **listed)
        km.sync()
        raw = out.read(np.uint16, offset + self.tokens * ot)
        rows = raw[offset:].reshape(self.tokens, ot)[:, :heads * oh].reshape(self.tokens, heads, oh)
        assert (raw[:offset] == 0x5A5A).all() and (rows[:, :, c.dim:] == 0x5A5A).all(), "written between the rows"
        values = from_bits(np.ascontiguousarray(rows[:, :, :c.dim]) if self.kind == BF16 else np.ascontiguousarray(rows[:, :, :c.dim]).view(np.float16), self.kind)
        return values.reshape(self.tokens, c.heads, self.group, c.dim).astype(np.float64), lse.read(np.float32, self.tokens * heads).reshape(self.tokens, c.heads, self.group).astype(np.float64)

    def check(self, **how):
        call = {k: how.pop(k) for k in ("gaps", "out_gaps", "offset") if k in how}
        got, lse = self.attend(**how, **call)
        want, want_lse, off, lse_off = self.expected(**how)
        empty = np.isneginf(want_lse)
        assert np.array_equal(np.isneginf(lse), empty) and not np.any(got[empty])
        assert np.all(np.abs(got - want) <= off), (np.abs(got - want) / np.maximum(off, 1e-300)).max()
        far = np.abs(lse[~empty] - want_lse[~empty])
        assert np.all(far <= lse_off[~empty]), (far / lse_off[~empty]).max()
        return got, lse


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("heads,group,dim,page,lengths", [
    (1, 1, 32, 16, [1]), (2, 4, 64, 32, [1, 15, 16, 17, 0, 63]), (2, 8, 128, 64, [64, 65, 127, 300]), (1, 16, 96, 256, [255, 257]), (3, 3, 160, 16, [200, 7]),
    (1, 17, 192, 128, [130]), (2, 5, 224, 64, [77, 500]), (1, 2, 256, 64, [1000, 3]), (1, 40, 64, 16, [90]), (4, 1, 128, 16, [33, 1500])])
def test_single_queries(km, gpu, kind, heads, group, dim, page, lengths):
    rng = np.random.default_rng(dim + group)
    c = Cache(km, rng, heads, dim, page, sum(-(-n // page) for n in lengths) + 2)
    Queries(km, rng, c, lengths, [1] * len(lengths), group, kind).fill(rng, kind).check()


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,group,dim,page,lengths,counts", [
    (2, 2, 64, 16, [40, 5, 1], [3, 5, 1]), (1, 6, 96, 64, [70, 130], [5, 3]), (1, 4, 128, 32, [20, 200], [16, 16]),      # up to 64 rows of a head
    (1, 8, 64, 64, [300, 64], [33, 20]), (2, 3, 128, 16, [100, 400], [100, 1]), (1, 1, 32, 16, [333], [333]),            # more: 256 rows a work-group
    (1, 5, 256, 128, [150], [60]), (1, 2, 160, 64, [129], [129]), (1, 4, 192, 256, [300], [66]), (1, 1, 224, 64, [70], [70])])
def test_several_queries(km, gpu, kind, causal, heads, group, dim, page, lengths, counts):
    rng = np.random.default_rng(dim + sum(counts))
    c = Cache(km, rng, heads, dim, page, sum(-(-n // page) for n in lengths) + 2)
    Queries(km, rng, c, lengths, counts, group, kind).fill(rng).check(causal=causal)


@pytest.mark.parametrize("group,counts", [(4, [1, 1]), (2, [40, 36])])
def test_tokens_in_parts(km, gpu, group, counts):
    """Long enough for parts of the tokens that are joined: by the last work-group, and by a kernel. Again, and again: the counters of the parts start from zero each time."""
    rng = np.random.default_rng(1)
    c = Cache(km, rng, 1, 64, 64, 200)
    s = Queries(km, rng, c, [9000, 3100], counts, group, BF16).fill(rng)
    first = s.check()
    for _ in range(3):
        again = s.attend()
        assert np.array_equal(first[0], again[0]) and np.array_equal(first[1], again[1])


SEVENTY = [2500 if s == 67 else 5 + s for s in range(70)]


@pytest.mark.parametrize("heads,group,dim,page,lengths,counts", [
    (2, 3, 96, 64, [3000, 500, 0, 64, 1], [30, 90, 5, 1, 3]),                              # a sequence much longer than the others
    (1, 4, 128, 16, [700, 1500], [300, 20]), (2, 1, 64, 32, [2000, 30, 900], [70, 2, 270]),  # some 256 rows of one, none of the other
    (2, 1, 32, 64, SEVENTY, [1 + s % 3 if s else 80 for s in range(70)]),                  # more than 64 sequences
    (3, 2, 256, 128, [500, 400], [40, 33]),                                                # all short: whole units
    (4, 1, 96, 16, [20 + s for s in range(70)], [66 if s == 9 else 1 for s in range(70)])])  # and more of them than work-groups
def test_lengths_far_below_what_the_batch_allows(km, gpu, heads, group, dim, page, lengths, counts):
    """The host knows the longest length that may come; what there is is divided on the device."""
    rng = np.random.default_rng(dim + len(lengths))
    c = Cache(km, rng, heads, dim, page, sum(-(-n // page) for n in lengths) + 2)
    tiles = -(-65536 // (heads * len(lengths)))
    s = Queries(km, rng, c, lengths, counts, group, BF16, extra=64 * tiles // page).fill(rng)
    s.batch = km.Cache4Batch(len(lengths), heads * group, s.tokens, max(counts), 64 * tiles, device(km, s.starts), device(km, np.int32(lengths)), device(km, s.table), s.table.shape[1])
    first = s.check()
    again = s.attend()
    assert np.array_equal(first[0], again[0]) and np.array_equal(first[1], again[1])


@pytest.mark.parametrize("counts", [[4, 9, 2], [70, 90, 80]])
def test_more_queries_than_tokens_and_empty_sequences(km, gpu, counts):
    """The first queries of a sequence that holds fewer tokens than it has queries see nothing: zeros and minus infinity."""
    rng = np.random.default_rng(2)
    c = Cache(km, rng, 2, 64, 16, 8)
    s = Queries(km, rng, c, [2, 0, 1], counts, 2, F16).fill(rng)
    got, lse = s.check()
    assert np.isneginf(lse[0]).all() and np.isneginf(lse[counts[0]:counts[0] + counts[1]]).all() and np.isfinite(lse[counts[0] - 1]).all()


@pytest.mark.parametrize("counts", [[1, 1], [40, 40]])
def test_strides_and_odd_addresses(km, gpu, counts):
    rng = np.random.default_rng(3)
    c = Cache(km, rng, 2, 96, 32, 10)
    s = Queries(km, rng, c, [100, 41], counts, 3, BF16).fill(rng)
    straight = s.check()
    for how in (dict(gaps=(8, 32), out_gaps=(16, 8), offset=8), dict(gaps=(1, 2), out_gaps=(3, 1), offset=1)):
        other = s.check(**how)
        assert np.array_equal(straight[0], other[0]) and np.array_equal(straight[1], other[1])


@pytest.mark.parametrize("counts", [[1], [70]])
@pytest.mark.parametrize("scale", [0.0, -0.3, 1e-6, 4.0])
def test_scales(km, gpu, counts, scale):
    rng = np.random.default_rng(4)
    c = Cache(km, rng, 1, 64, 64, 5)
    Queries(km, rng, c, [200], counts, 2, F16, loud=0.5).fill(rng).check(scale=scale)


@pytest.mark.parametrize("counts", [[1], [70]])
@pytest.mark.parametrize("kind,loud", [(BF16, 1e30), (BF16, 1e-30), (F16, 1e-5), (F16, 1e4)])
def test_large_and_small_queries(km, gpu, counts, kind, loud):
    rng = np.random.default_rng(5)
    c = Cache(km, rng, 1, 64, 64, 5)
    s = Queries(km, rng, c, [150], counts, 2, kind, loud=loud).fill(rng)
    s.check(scale=0.2 / loud)


@pytest.mark.parametrize("counts", [[1, 1], [70, 50]])
def test_pages_that_are_not_there_and_pages_shared(km, gpu, counts):
    """Entries of the table outside the cache are left out; two sequences may look at the same pages."""
    rng = np.random.default_rng(6)
    c = Cache(km, rng, 1, 64, 16, 20)
    s = Queries(km, rng, c, [150, 120], counts, 2, F16).fill(rng)
    s.table[1, :4] = s.table[0, :4]
    s.table[0, 5], s.table[0, 2], s.table[1, 6] = -1, 20, 1 << 30
    s.batch = km.Cache4Batch(2, 2, s.tokens, max(counts), 150, device(km, s.starts), device(km, np.int32(s.lengths)), device(km, s.table), s.table.shape[1])
    s.check()


def test_lengths_beyond_the_table_are_cut(km, gpu):
    rng = np.random.default_rng(7)
    c = Cache(km, rng, 1, 32, 16, 4)
    s = Queries(km, rng, c, [64], [1], 1, F16, extra=0).fill(rng)
    full = s.check()
    s.batch = km.Cache4Batch(1, 1, 1, 1, 1 << 30, device(km, s.starts), device(km, np.int32([(1 << 31) - 1])), device(km, s.table), 4)
    assert np.array_equal(s.attend()[0], full[0])
    s.batch = km.Cache4Batch(1, 1, 1, 1, 1 << 30, device(km, s.starts), device(km, np.int32([-5])), device(km, s.table), 4)
    got, lse = s.attend()
    assert not np.any(got) and np.isneginf(lse).all()


def test_nan_stays_in_its_row(km, gpu):
    rng = np.random.default_rng(9)
    c = Cache(km, rng, 2, 64, 32, 6)
    s = Queries(km, rng, c, [100, 30], [1, 1], 4, BF16).fill(rng)
    clean = s.attend()
    s.q[1, 0, 2, 5] = np.nan
    got, lse = s.attend()
    assert np.isnan(got[1, 0, 2]).all()
    got[1, 0, 2], lse[1, 0, 2] = clean[0][1, 0, 2], clean[1][1, 0, 2]
    assert np.array_equal(got, clean[0]) and np.array_equal(lse, clean[1])


# ---------------------------------------------------------------- chosen pages -------------------

def bounds_of(c, page, tokens):
    """(largest, smallest in 8 bits, scale) of a page, (heads, dim) each."""
    rows = c.k[page * c.page:page * c.page + tokens]
    hi, lo = (rows.max(0), rows.min(0)) if tokens else (np.zeros((c.heads, c.dim), np.float32),) * 2
    top = np.maximum(np.abs(hi), np.abs(lo)).max(-1, keepdims=True)
    with np.errstate(divide="ignore"):
        by = np.where(top > 0, np.float32(1) / top * np.float32(127), np.float32(0))
    return np.clip(np.ceil(hi * by), -127, 127).astype(np.int8), np.clip(np.floor(lo * by), -127, 127).astype(np.int8), (top[:, 0] / np.float32(127))


def kept_bounds(c):
    n = c.pages * c.heads
    raw = c.bounds.read(np.uint8, n * (2 * c.dim + 4))
    return raw[:n * 2 * c.dim].view(np.int8).reshape(c.pages, c.heads, 2 * c.dim), raw[n * 2 * c.dim:].view(np.float32).reshape(c.pages, c.heads)


def bound_all(s):
    """Bounds of all pages of all sequences, and what they are to be."""
    c, km = s.c, s.km
    pages, counts = [], []
    for b, n in enumerate(s.lengths):
        for e in range(-(-n // c.page)):
            pages.append(int(s.table[b, e]))
            counts.append(min(c.page, n - e * c.page))
    c.dev.bound(device(km, np.int32(pages)), device(km, np.int32(counts)), len(pages))
    km.sync()
    want = {p: bounds_of(c, p, n) for p, n in zip(pages, counts)}
    return want


def choice(s, want, top, first, last, causal):
    c = s.c
    out = np.full((s.tokens, c.heads, top), -1, np.int64)
    for b in range(len(s.lengths)):
        for i in range(s.counts[b]):
            t, n = s.starts[b] + i, -(-s.sees(b, i, causal) // c.page)
            for h in range(c.heads):
                q = s.q[t, h]
                m = np.abs(q).max()
                by = np.float32(1) / np.float32(m) * np.float32(127) if m > 0 else np.float32(0)
                q8 = np.clip(np.rint(q * by), -127, 127).astype(np.int64)
                score = np.empty(n, np.float32)
                for e in range(n):
                    if s.table[b, e] < 0 or s.table[b, e] >= c.pages:
                        score[e] = -np.inf
                    else:
                        hi, lo, scale = want[int(s.table[b, e])]
                        score[e] = np.float32(np.maximum(q8 * hi[h].astype(np.int64), q8 * lo[h].astype(np.int64)).sum(-1).max()) * scale[h]
                at = np.arange(n)
                score[(at < first) | (at + last >= n)] = np.inf
                best = np.sort(np.argsort(-score, kind="stable")[:top])
                out[t, h, :len(best)] = best
    return out


def select(s, top, first, last, causal=True):
    km = s.km
    bits = device(km, to_bits(s.q, s.kind))
    chosen = device(km, np.full(s.tokens * s.c.heads * top + 8, 12345, np.int32))
    s.c.dev.select(s.batch, s.kind, bits, chosen, top, first, last, causal)
    km.sync()
    raw = chosen.read(np.int32, s.tokens * s.c.heads * top + 8)
    assert (raw[-8:] == 12345).all()
    return raw[:-8].reshape(s.tokens, s.c.heads, top)


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("heads,group,dim,page,lengths,counts,top,first,last", [
    (1, 1, 32, 16, [100], [1], 3, 1, 1), (2, 4, 64, 16, [500, 17, 1], [1, 1, 1], 6, 1, 1), (1, 8, 128, 64, [700, 300], [1, 3], 4, 0, 2),
    (2, 3, 96, 32, [400], [9], 5, 1, 1), (1, 20, 64, 16, [300], [2], 7, 2, 0), (1, 16, 160, 16, [200, 90], [1, 2], 4, 1, 1), (1, 2, 192, 16, [130], [130], 3, 1, 1),
    (1, 5, 224, 128, [600], [1], 2, 0, 0), (1, 4, 256, 256, [2000], [5], 3, 1, 1), (1, 1, 64, 16, [9000], [1], 40, 1, 1), (2, 2, 32, 16, [14000, 9000], [1, 2], 16, 1, 1),
    (1, 33, 32, 16, [13000], [1], 30, 1, 1)])
def test_bounds_choice_and_attention_to_it(km, gpu, kind, heads, group, dim, page, lengths, counts, top, first, last):
    """Few pages and many (from 769 on scores and choice are two kernels), queries that see fewer pages than they may choose, more than 16 query heads."""
    rng = np.random.default_rng(dim + top)
    c = Cache(km, rng, heads, dim, page, sum(-(-n // page) for n in lengths) + 2)
    s = Queries(km, rng, c, lengths, counts, group, kind).fill(rng)
    want = bound_all(s)
    eight, scales = kept_bounds(c)
    for p, (hi, lo, scale) in want.items():
        assert np.array_equal(eight[p], np.concatenate([hi, lo], -1)) and np.array_equal(scales[p], scale)
    chosen = select(s, top, first, last)
    assert np.array_equal(chosen, choice(s, want, top, first, last, True))
    s.check(chosen=chosen)


def test_all_pages_chosen_is_all_attention(km, gpu):
    rng = np.random.default_rng(11)
    c = Cache(km, rng, 2, 64, 32, 12)
    s = Queries(km, rng, c, [200, 100], [2, 1], 4, F16).fill(rng)
    bound_all(s)
    chosen = select(s, 9, 1, 1)
    got, want = s.check(chosen=chosen), s.attend()
    assert np.abs(got[0] - want[0]).max() < 4 * UNIT[F16] * np.abs(want[0]).max()


def test_choice_without_causality_and_equal_scores(km, gpu):
    """Pages written alike have equal scores: the first ones are taken. Pages that are not there come last."""
    rng = np.random.default_rng(12)
    c = Cache(km, rng, 1, 32, 16, 20)
    s = Queries(km, rng, c, [256], [4], 2, BF16)
    rows = ordinary(rng, 16, 1, 32)
    for p in s.table[0, :16]:
        c.write(F32, *rows, p * 16 + np.arange(16))
    want = bound_all(s)
    assert np.array_equal(select(s, 5, 0, 1, causal=False), np.broadcast_to([0, 1, 2, 3, 15], (4, 1, 5)))
    s.table[0, 1], s.table[0, 3] = -1, 99
    s.batch = km.Cache4Batch(1, 2, 4, 4, 256, device(km, s.starts), device(km, np.int32([256])), device(km, s.table), s.table.shape[1])
    assert np.array_equal(select(s, 5, 0, 0, causal=False), np.broadcast_to([0, 2, 4, 5, 6], (4, 1, 5)))
    assert np.array_equal(select(s, 16, 0, 0, causal=False), np.broadcast_to(np.arange(16), (4, 1, 16)))
    assert np.array_equal(choice(s, want, 5, 0, 0, False), np.broadcast_to([0, 2, 4, 5, 6], (4, 1, 5)))


def test_bounds_of_few_tokens_and_of_pages_that_are_not_there(km, gpu):
    rng = np.random.default_rng(13)
    c = Cache(km, rng, 2, 96, 64, 4)
    c.write(F16, *ordinary(rng, 256, 2, 96), np.arange(256))
    pages, counts = [2, -1, 0, 4, 3, 1 << 30], [1, 5, 0, 9, 300, 1]
    c.dev.bound(device(km, np.int32(pages)), device(km, np.int32(counts)), 6)
    km.sync()
    eight, scales = kept_bounds(c)
    for p, n in ((2, 1), (0, 0), (3, 64)):
        hi, lo, scale = bounds_of(c, p, n)
        assert np.array_equal(eight[p], np.concatenate([hi, lo], -1)) and np.array_equal(scales[p], scale)
    assert (eight[1] == -1).all()  # nobody asked for it


# ---------------------------------------------------------------- around the kernels -------------

def test_recorded_steps(km, gpu):
    """A recorded step replayed, the program's own calls between: every replay as the call itself."""
    rng = np.random.default_rng(14)
    c = Cache(km, rng, 2, 64, 64, 120)
    s = Queries(km, rng, c, [4000, 2500], [1, 1], 4, BF16).fill(rng)
    bound_all(s)
    s.c.dev.reserve(s.batch, 8)
    q, out = device(km, to_bits(s.q, BF16)), device(km, np.zeros(s.tokens * 8 * 64, np.uint16))
    chosen, sparse = device(km, np.zeros(s.tokens * 2 * 8, np.int32)), device(km, np.zeros(s.tokens * 8 * 64, np.uint16))

    def step():
        c.dev.select(s.batch, BF16, q, chosen, 8)
        c.dev.attend(s.batch, BF16, q, sparse, s.scale, chosen=chosen, top=8)
        c.dev.attend(s.batch, BF16, q, out, s.scale)

    def results():
        km.sync()
        return out.read(np.uint16, s.tokens * 512), sparse.read(np.uint16, s.tokens * 512), chosen.read(np.int32, s.tokens * 16)

    step()
    want = results()
    with km.Graph() as g:
        step()
    for _ in range(4):
        for b in (out, sparse, chosen):
            b.zero()
        g.launch()
        assert all(np.array_equal(a, b) for a, b in zip(results(), want))
        step()
        km.sync()
    # other queries in the same buffer
    s.q = from_bits(to_bits(rng.normal(size=s.q.shape), BF16), BF16)
    q.write(to_bits(s.q, BF16))
    g.launch()
    replayed = results()
    step()
    assert all(np.array_equal(a, b) for a, b in zip(results(), replayed)) and not np.array_equal(replayed[0], want[0])
    g.destroy()


def test_on_a_stream_of_the_callers(km, gpu):
    rng = np.random.default_rng(15)
    c = Cache(km, rng, 1, 64, 64, 80)
    s = Queries(km, rng, c, [5000], [1], 4, F16).fill(rng)
    want = s.attend()
    import ctypes
    hip = ctypes.CDLL(next(line.split()[-1] for line in open("/proc/self/maps") if "libamdhip64" in line))  # the runtime that the library runs on
    stream = ctypes.c_void_p()
    assert hip.hipStreamCreateWithFlags(ctypes.byref(stream), 1) == 0  # waits for no other stream
    km.check(km.hip_lib().kmx_set_stream(stream))
    try:
        for _ in range(3):
            got = s.attend()
            assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
    finally:
        km.sync()
        km.check(km.hip_lib().kmx_set_stream(None))
        assert hip.hipStreamDestroy(stream) == 0
    again = s.attend()
    assert np.array_equal(again[0], want[0])


def test_k_means_calls_keep_their_work_space(km, gpu):
    """The parts of the attention share the library's work space with the updates: an update between two calls, and the other way round."""
    rng = np.random.default_rng(16)
    c = Cache(km, rng, 1, 64, 64, 80)
    s = Queries(km, rng, c, [5000], [1], 4, F16).fill(rng)
    want = s.attend()
    data = np.float32(rng.normal(size=(20000, 16))).reshape(-1)
    alg = km.HipKMeansAlgorithm()
    alg.initialize(16, 50, 20000, 4, data, data[:50 * 16])
    alg.run(2)
    middle = alg.getMeans()
    got = s.attend()
    alg.reset(data[:50 * 16])
    alg.run(2)
    assert np.array_equal(got[0], want[0]) and np.array_equal(alg.getMeans(), middle)
    alg.cleanup()


def test_learned_levels_beat_even_ones(km, gpu):
    """The levels that k-means finds hold normal rows better than evenly spaced ones of the same number."""
    rng = np.random.default_rng(17)
    rows = np.float32(rng.standard_t(6, size=(4000, 1, 64)))
    learned = km.cache4_learn_levels(rows)
    assert learned.dtype == np.float16 and np.all(np.diff(learned) > 0)
    even = km.cache4_round_levels((np.arange(8) + 0.5) / 8)
    error = lambda lv: float(((held(rows, lv[None]) - rows) ** 2).mean())  # noqa: E731
    assert error(learned) < 0.9 * error(even)


def test_the_example(km, gpu):
    """The whole path: levels and layout learned by k-means, rows written, bounds, choice, attention. With the pages laid out by clusters the chosen
    ones come closer to attention to all rows than with the prompt's order."""
    import importlib.util
    import os
    spec = importlib.util.spec_from_file_location("cache4_decode", os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "cache4_decode.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    got = example.run(prompt=3000, steps=5, heads=2, group=4, dim=64, page=32, pages=16, say=lambda text: None)
    assert got["by clusters"]["sparse"] < got["prompt's order"]["sparse"]
    assert got["by clusters"]["whole"] < 0.2 and got["prompt's order"]["whole"] < 0.2
