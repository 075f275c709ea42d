"""How the attention over the 4-bit cache is launched and what room it takes (csrc/cache4_plan.h), on the host: batches that no test could allocate."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
UNITS = 256  # compute units of the card


def room(dim):
    """Bytes that the parts of many rows take at most: eight rounds of work-groups, two on a compute unit up to 64 channels."""
    return 4 * 8 * UNITS * (2 if dim <= 64 else 1) * 256 * (dim + 2)


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    folder = tmp_path_factory.mktemp("plan")
    src, lib = folder / "plan.cpp", folder / "libplan.so"
    src.write_text('#include "cache4_plan.h"\n'
                   'using namespace kmx;\n'
                   'extern "C" void plan(const uint32_t* s, uint64_t* out)\n'
                   "{ const Plan4 p = plan_attend4(Shape4{ s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], s[8] });\n"
                   "  out[0] = p.units; out[1] = p.row_tiles; out[2] = p.splits; out[3] = p.tiles_per_split; out[4] = p.many; out[5] = p.joined; out[6] = plan_floats(p, s[0]); }\n"
                   'extern "C" uint64_t most(const uint32_t* s) { return most_floats(Shape4{ s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], s[8] }); }\n')
    subprocess.check_call(["g++", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I", os.path.join(ROOT, "cuda-kmeans_amd", "csrc"), str(src), "-o", str(lib)])
    lib = ctypes.CDLL(str(lib))
    lib.most.restype = ctypes.c_uint64

    def call(dim, heads, group, sequences, queries, length, page=64, top=0, most=False):
        out = np.zeros(7, np.uint64)
        numbers = np.array([dim // 32, heads, group, sequences, queries, length, page.bit_length() - 1, top, UNITS], np.uint32)
        if most:
            return lib.most(numbers.ctypes.data_as(ctypes.c_void_p))
        lib.plan(numbers.ctypes.data_as(ctypes.c_void_p), out.ctypes.data_as(ctypes.c_void_p))
        return dict(zip(("units", "row_tiles", "splits", "tiles_per_split", "many", "joined", "floats"), (int(v) for v in out)))
    return call


def batches(seed, count):
    rng = np.random.default_rng(seed)
    spread = lambda low, high: int(round(np.exp(rng.uniform(np.log(low), np.log(high)))))  # noqa: E731
    for _ in range(count):
        yield dict(dim=32 * spread(1, 8), heads=spread(1, 64), group=spread(1, 64), sequences=spread(1, 5000), queries=spread(1, 60000) if rng.random() < 0.7 else 1,
                   length=spread(1, 2 ** 31 - 1), page=16 << int(rng.integers(0, 5)))


def test_a_piece_of_a_prompt_a_little_above_a_round_of_work_groups(plan):
    """131072 tokens, 64 heads on 8: 1024 queries are as many units as compute units; 1056 want parts, and take less than 0.6 GB."""
    for dim in (32, 64, 128, 256):
        assert plan(dim, 8, 8, 1, 1024, 131072)["floats"] == 0 or dim <= 64
        for queries in range(1025, 1400, 31):
            assert plan(dim, 8, 8, 1, queries, 131072)["floats"] * 4 <= room(dim) + 16 * 1024
    assert plan(128, 8, 8, 1, 1056, 131072)["splits"] >= 4 * 264  # still several parts
    assert plan(128, 8, 16, 1, 8300, 131072)["floats"] * 4 <= 300e6
    assert max(room(dim) for dim in range(32, 257, 32)) < 0.6e9


def test_room_of_any_batch(plan):
    for b in batches(1, 20000):
        p = plan(**b)
        words = 2 * p["units"]
        assert 4 * p["floats"] <= room(b["dim"]) + 4 * words, b
        for top in (1, 8, 100):
            assert 4 * plan(**b, top=top)["floats"] <= room(b["dim"])


def test_parts_cover_all_tokens(plan):
    """Every tile of 64 tokens is in a part, none of which is empty at the full length; shares count work-groups that the chip holds."""
    for b in batches(2, 20000):
        for top in (0, 3, 64):
            p = plan(**b, top=top)
            if p["units"] >= 1 << 23:
                assert p["floats"] == 0
                continue
            rows = b["queries"] * b["group"]
            want = b["queries"] * -(-b["group"] // 16) if top else -(-rows // 256) if rows > 64 else -(-rows // 16)
            assert p["row_tiles"] == want and p["units"] == b["sequences"] * b["heads"] * want and p["many"] == (not top and rows > 64)
            tiles = -(-(min(top, -(-b["length"] // b["page"])) * b["page"] if top else b["length"]) // 64)
            if p["many"] and p["tiles_per_split"] == 0:
                assert p["splits"] in (UNITS, 2 * UNITS) and p["joined"]
                assert p["floats"] == 2 * p["splits"] * 256 * (b["dim"] + 2) + 2 * p["units"]
                continue
            parts = p["splits"] // p["units"] if p["many"] else p["splits"]
            assert p["tiles_per_split"] * parts >= tiles
            if p["many"]:
                assert p["splits"] == parts * p["units"] and p["joined"] == (parts > 1)
                assert p["floats"] == (p["splits"] * 256 * (b["dim"] + 2) + 2 * p["units"] if parts > 1 else 0)
            else:
                assert p["tiles_per_split"] * (parts - 1) < tiles and p["tiles_per_split"] % 4 == 0 and parts <= 128
                assert p["floats"] == (p["units"] * parts * 16 * (b["dim"] + 2) if parts > 1 else 0)


def test_lists_longer_than_any_sequence(plan):
    """As many tokens as 32 bits do not count if the lists were full: what a sequence can have decides, in as many parts as there are work-groups for."""
    for page in (16, 64, 256):
        for top in ((1 << 30) - 1, 1 << 30, (1 << 30) + 1, (1 << 32) - 1):
            for length in (1, 9000, 2 ** 31 - 1):
                p, pages = plan(64, 1, 2, 1, 1, length, page, top), -(-length // page)
                assert p["splits"] * p["tiles_per_split"] >= -(-pages * page // 64)
                assert p == plan(64, 1, 2, 1, 1, length, page, pages)
                assert (p["floats"] > 0) == (p["splits"] > 1) == (length > 1000)


def test_room_for_a_batch_is_room_for_smaller_ones(plan):
    """Fewer units have more parts: 64 sequences of 8 heads need nothing, 63 do. What is reserved for a batch holds for all that are no larger, and is not
    more than the largest of them could take by far: 1024 parts of 16 rows, eight rounds of parts of 256."""
    full, fewer = (plan(128, 8, 4, n, 1, 8192) for n in (64, 63))
    assert full["floats"] == 0 and fewer["floats"] > 0 and plan(128, 8, 4, 64, 1, 8192, most=True) >= fewer["floats"]
    rng = np.random.default_rng(4)
    for b in batches(3, 20000):
        top = int(rng.integers(1, 200)) if rng.random() < 0.5 else 0
        most = plan(**b, top=top, most=True)
        assert most <= max(4 * UNITS * 16 * (b["dim"] + 2), 8 * UNITS * (2 if b["dim"] <= 64 else 1) * (256 * (b["dim"] + 2) + 1))
        for _ in range(8):
            less = dict(b, **{name: int(np.ceil(b[name] * rng.random() ** rng.integers(0, 4))) or 1 for name in ("sequences", "queries", "length")})
            assert plan(**less)["floats"] <= most, (b, less)
            if top:
                assert plan(**less, top=int(rng.integers(1, top + 1)))["floats"] <= most, (b, less, top)
    for sequences in range(1, 70):
        for queries in (1, 5, 17, 64, 300, 1056):
            for length in (1, 300, 5000, 131072):
                assert plan(128, 8, 4, sequences, queries, length)["floats"] <= plan(128, 8, 4, 70, 1056, 131072, most=True)
