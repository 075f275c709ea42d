"""Rotary positions on the GPU (csrc/rotary.hip) against their definition: angles by whole numbers, the rest in 64 bits (-m gpu)."""
import numpy as np
import pytest

from test_gpu_cache4 import BF16, F16, F32, UNIT, device, from_bits, to_bits

pytestmark = pytest.mark.gpu

ROUNDING = {F32: 2.0 ** -24, **UNIT}


def bits_type(kind):
    return {F32: np.float32, F16: np.float16, BF16: np.uint16}[kind]


def rotated(x, positions, turns, channels, halves, inverse, gain):
    """x: tokens x heads x dim. (result, how far it may be off before it is rounded to its type)"""
    x, half = x.astype(np.float64), channels // 2
    whole = [[(int(p) * int(f)) % 2 ** 64 for f in turns] for p in positions]
    angle = 2 * np.pi * (np.array(whole, dtype=np.float64).reshape(len(positions), half) / 2.0 ** 64)
    c, s = gain * np.cos(angle)[:, None], (-gain if inverse else gain) * np.sin(angle)[:, None]
    i = np.arange(half)
    a, b = (i, i + half) if halves else (2 * i, 2 * i + 1)
    out, off = x.copy(), np.zeros_like(x)
    out[..., a], out[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    # sine and cosine: the angle to 2^-24 of at most a quarter turn twice and to 2^-32 of a turn, the series to 2^-25, its sum rounded: 2^-22 in all; then the gain, two
    # products and their sum, each to 2^-24
    off[..., a] = off[..., b] = 2.0 ** -21 * abs(gain) * (np.abs(x[..., a]) + np.abs(x[..., b]))
    return out, off


def check(km, rng, kind, tokens, heads, dim, channels, halves=True, inverse=False, gain=1.0, positions=None, turns=None, gaps=(0, 0), out_gaps=(0, 0), offset=0, in_place=False, loud=1.0):
    """heads: of each set."""
    turns = km.rotary_turns(channels) if turns is None else turns
    positions = rng.integers(0, 131072, tokens) if positions is None else np.asarray(positions)
    sets, held = [], []
    for n in heads:
        x = from_bits(to_bits(rng.normal(size=(tokens, n, dim)) * loud, kind), kind)
        hs, ohs = dim + gaps[0], dim + out_gaps[0]
        ts, ots = n * hs + gaps[1], n * ohs + out_gaps[1]
        flat = np.full(offset + tokens * ts, 7, np.float32)
        for t in range(tokens):
            flat[offset + t * ts:][:n * hs].reshape(n, hs)[:, :dim] = x[t]
        src = device(km, to_bits(flat, kind))
        item = 4 if kind == F32 else 2
        pattern = np.full((offset + tokens * ots) * item, 0x5A, np.uint8)
        dst = src if in_place else device(km, pattern)
        view = lambda b: km.DeviceView(b.ptr.value + offset * item, 0)  # noqa: E731
        sets.append(km.RotaryRows(view(src), n, None if in_place else view(dst), ts, hs, ots, ohs))
        held.append((x, src, dst, ts if in_place else ots, hs if in_place else ohs))
    turn_buf, position_buf = device(km, turns), device(km, positions.astype(np.int32))
    km.rotary(kind, sets, tokens, dim, turn_buf, position_buf, channels=channels, halves=halves, inverse=inverse, gain=gain)
    km.sync()
    results = []
    for (x, src, dst, ts, hs), n in zip(held, heads):
        raw = dst.read(bits_type(kind), offset + tokens * ts)
        rows = raw[offset:].reshape(tokens, ts)[:, :n * hs].reshape(tokens, n, hs)
        if in_place:
            assert np.all(from_bits(np.ascontiguousarray(rows[..., dim:]), kind) == 7) and np.all(from_bits(raw[:offset], kind) == 7), "written between the rows"
        else:
            assert (np.ascontiguousarray(rows[..., dim:]).view(np.uint8) == 0x5A).all() and (raw[:offset].view(np.uint8) == 0x5A).all(), "written between the rows"
        got = from_bits(np.ascontiguousarray(rows[..., :dim]), kind)
        want, off = rotated(x, positions, turns, channels, halves, inverse, gain)
        assert np.array_equal(got[..., channels:], x[..., channels:])
        far = np.abs(got.astype(np.float64) - want)
        bound = off * (1 + ROUNDING[kind]) + ROUNDING[kind] * np.abs(want) + (2.0 ** -25 if kind == F16 else 2.0 ** -126)  # (of the smallest numbers the type has fewer bits)
        assert np.all(far <= bound), (far / bound).max()
        results.append(got)
    return results


@pytest.mark.parametrize("kind", [F32, F16, BF16])
@pytest.mark.parametrize("halves", [True, False])
@pytest.mark.parametrize("tokens,heads,dim,channels", [(1, (1,), 2, 2), (3, (2, 1), 32, 32), (5, (4, 2), 64, 16), (2, (3,), 96, 64), (33, (8, 2, 1), 128, 128), (7, (5, 1), 80, 80), (4, (3, 3), 72, 20),
                                                    (3, (2,), 31, 14), (2, (1, 2), 256, 96), (3, (2,), 40, 0), (9, (1, 1, 1, 1), 24, 24)])
def test_rows_are_rotated_as_defined(km, gpu, kind, halves, tokens, heads, dim, channels):
    rng = np.random.default_rng(dim + channels)
    for in_place in (False, True):
        there = check(km, rng, kind, tokens, heads, dim, channels, halves, in_place=in_place)
        assert len(there) == len(heads)


@pytest.mark.parametrize("kind", [F32, BF16])
def test_far_positions(km, gpu, kind):
    """Angles of positions that 32 bits hold, either sign, and frequencies of whole turns, halves and quarters of them."""
    rng = np.random.default_rng(1)
    positions = [0, 1, -1, 2 ** 31 - 1, -2 ** 31, 2 ** 24 + 1, 1000003, -1000003, 65536, 7]
    check(km, rng, kind, len(positions), (2,), 128, 128, positions=positions, turns=km.rotary_turns(128, 500000.0, 8.0, 8192.0, 1.0, 4.0))
    turns = np.array([0, 1 << 63, 1 << 62, (1 << 62) + 1, (1 << 61) - 1, 1 << 61, 2 ** 64 - 1, 3 << 61], np.uint64)
    check(km, rng, kind, len(positions), (1,), 16, 16, positions=positions, turns=turns)
    check(km, rng, kind, len(positions), (1,), 16, 16, positions=positions, turns=turns, halves=False, inverse=True)


def test_the_series_over_a_whole_turn(km, gpu):
    """Sine and cosine themselves, at all angles: rows of (1, 0)."""
    n = 1 << 14
    turns = np.array([(1 << 50) + 977], np.uint64)
    rows = device(km, np.tile(np.float32([1, 0]), (n, 1)))
    km.rotary(km.TYPE_F32, [km.RotaryRows(rows, 1)], n, 2, device(km, turns), device(km, np.arange(n, dtype=np.int32)))
    km.sync()
    got = rows.read(np.float32, 2 * n).reshape(n, 2).astype(np.float64)
    angle = 2 * np.pi * (np.arange(n) * float(turns[0]) / 2.0 ** 64)
    assert np.abs(got - np.stack([np.cos(angle), np.sin(angle)], -1)).max() <= 2.0 ** -22


@pytest.mark.parametrize("kind", [F32, F16, BF16])
def test_there_and_back(km, gpu, kind):
    """The inverse takes rows back, and is the transpose: <g, R x> = <R^-1 g, x>, which is what a gradient takes."""
    rng = np.random.default_rng(2)
    tokens, heads, dim, channels = 40, 6, 128, 96
    x, g = (from_bits(to_bits(rng.normal(size=(tokens, heads, dim)), kind), kind) for _ in range(2))
    turns, positions = device(km, km.rotary_turns(channels)), device(km, rng.integers(0, 100000, tokens).astype(np.int32))

    def run(rows, inverse):
        b = device(km, to_bits(rows, kind))
        km.rotary(kind, [km.RotaryRows(b, heads)], tokens, dim, turns, positions, channels=channels, halves=False, inverse=inverse)
        km.sync()
        return from_bits(b.read(bits_type(kind), tokens * heads * dim), kind).reshape(x.shape)

    there, back = run(x, False), run(g, True)
    size = np.abs(x[..., 0:channels:2]) + np.abs(x[..., 1:channels:2])
    size = np.concatenate([np.repeat(size, 2, -1), np.abs(x[..., channels:])], -1)
    again = run(there, True)
    assert np.all(np.abs(again.astype(np.float64) - x) <= 4 * (ROUNDING[kind] + 2.0 ** -21) * size)  # two roundings of a and b each
    left, right = (g.astype(np.float64) * there).sum(), (back.astype(np.float64) * x).sum()
    assert abs(left - right) <= (ROUNDING[kind] + 2.0 ** -21) * 2 * (np.abs(g[..., :channels]).sum() * 2 * np.abs(x).max())


def test_gradients_by_differences(km, gpu):
    """d/dx of sum(w R(x)) is R^-1(w): against differences of the forward call. The rotation is linear, so a step of 1 is as good as any."""
    rng = np.random.default_rng(3)
    tokens, dim = 5, 32
    w = np.float32(rng.normal(size=(tokens, 1, dim)))
    turns, positions = device(km, km.rotary_turns(dim)), device(km, np.int32([0, 1, 100, 5000, 131071]))

    def run(rows, inverse):
        b = device(km, np.float32(rows))
        km.rotary(F32, [km.RotaryRows(b, 1)], tokens, dim, turns, positions, halves=True, inverse=inverse, gain=1.25)
        km.sync()
        return b.read(np.float32, tokens * dim).reshape(tokens, 1, dim).astype(np.float64)

    grad = run(w, True)
    for c in range(dim):
        step = np.zeros((tokens, 1, dim), np.float32)
        step[..., c] = 1
        assert np.all(np.abs((w * run(step, False)).sum(-1)[:, 0] - grad[:, 0, c]) <= 2.0 ** -20 * 1.25 * 2 * np.abs(w).max())


@pytest.mark.parametrize("kind", [F32, F16, BF16])
def test_strides_and_odd_addresses(km, gpu, kind):
    for how in (dict(gaps=(8, 16), out_gaps=(16, 32), offset=8), dict(gaps=(1, 3), out_gaps=(5, 2), offset=3), dict(gaps=(24, 8), offset=16, in_place=True), dict(gaps=(3, 1), offset=1, in_place=True)):
        for halves in (True, False):
            check(km, np.random.default_rng(4), kind, 21, (5, 2), 64, 48, halves, **how)


def test_gain_large_numbers_and_nan(km, gpu):
    rng = np.random.default_rng(5)
    check(km, rng, BF16, 10, (2,), 64, 64, gain=-1.3466)
    check(km, rng, F32, 10, (2,), 64, 64, gain=0.0)
    check(km, rng, F32, 10, (2,), 64, 64, loud=1e37)
    check(km, rng, BF16, 10, (2,), 64, 64, loud=1e-37)
    x = np.float32(rng.normal(size=(2, 1, 16)))
    x[0, 0, 3], x[1, 0, 12] = np.nan, np.inf
    b = device(km, x)
    km.rotary(F32, [km.RotaryRows(b, 1)], 2, 16, device(km, km.rotary_turns(16)), device(km, np.int32([5, 9])))
    km.sync()
    got = b.read(np.float32, 32).reshape(2, 16)
    bad = np.zeros((2, 16), bool)
    bad[0, [3, 11]] = bad[1, [4, 12]] = True
    assert np.array_equal(~np.isfinite(got), bad), "what is no number stays in its pair"


def test_many_tokens(km, gpu):
    """As many heads a lane as there may be, and more work-groups than fit the chip."""
    rng = np.random.default_rng(6)
    tokens, heads, dim = 6000, 37, 128
    x = from_bits(to_bits(rng.normal(size=(tokens, heads, dim)), BF16), BF16)
    rows, out = device(km, to_bits(x, BF16)), km.DeviceBuffer(2 * x.size)
    turns, positions = km.rotary_turns(dim), np.arange(tokens)
    km.rotary(BF16, [km.RotaryRows(rows, heads, out)], tokens, dim, device(km, turns), device(km, positions.astype(np.int32)))
    km.sync()
    got = from_bits(out.read(np.uint16, x.size), BF16).reshape(x.shape)
    some = np.concatenate([np.arange(20), rng.integers(0, tokens, 200), [tokens - 1]])
    want, off = rotated(x[some], positions[some], turns, dim, True, False, 1.0)
    assert np.all(np.abs(got[some] - want) <= off * 1.01 + UNIT[BF16] * np.abs(want) + 2.0 ** -126)
    size = np.sqrt((x.astype(np.float64) ** 2).sum(-1))
    assert np.abs(np.sqrt((got.astype(np.float64) ** 2).sum(-1)) / size - 1).max() < 2.0 ** -8  # lengths of all rows
