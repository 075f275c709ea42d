"""The keys by which pages are chosen (csrc/cache4_keys.h), on the host: whatever the bounds hold, no score has the key of a page that is always
taken, so a list has room for all pages with that key."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FORCED, MISSING = 0xFF800000, 0x007FFFFF
LARGEST = np.finfo(np.float32).max


@pytest.fixture(scope="module")
def key(tmp_path_factory):
    folder = tmp_path_factory.mktemp("keys")
    src, lib = folder / "keys.cpp", folder / "libkeys.so"
    src.write_text('#include "cache4_keys.h"\n'
                   'extern "C" uint32_t key(int forced, int known, int best, float scale) { return kmx::page_key(forced != 0, known != 0, best, scale); }\n'
                   'extern "C" uint32_t ordered(float v) { return kmx::ordered(v); }\n')
    subprocess.check_call(["g++", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I", os.path.join(ROOT, "cuda-kmeans_amd", "csrc"), str(src), "-o", str(lib)])
    lib = ctypes.CDLL(str(lib))
    lib.key.restype, lib.key.argtypes = ctypes.c_uint32, [ctypes.c_int] * 3 + [ctypes.c_float]
    lib.ordered.restype, lib.ordered.argtypes = ctypes.c_uint32, [ctypes.c_float]
    return lib


def test_no_score_has_the_key_of_a_page_that_is_always_taken(key):
    rng = np.random.default_rng(1)
    scales = np.concatenate([rng.integers(0, 1 << 32, 4000, dtype=np.uint32).view(np.float32),
                             np.float32([0, -0.0, 1e-45, 1, 1e34, 1e38, LARGEST, np.inf, -1e38, -LARGEST, -np.inf, np.nan, -np.nan])])
    for best in (1, 7, 127 * 127 * 256, 0, -1, -127 * 127 * 256, 127 * 128 * 256):
        with np.errstate(over="ignore", invalid="ignore"):
            score = np.float32(best) * scales
        want = np.where(np.isnan(score), -LARGEST, np.clip(score, -LARGEST, LARGEST))
        for scale, w in zip(scales, want):
            k = key.key(0, 1, best, float(scale))
            assert MISSING < k < FORCED and k == key.ordered(float(w + np.float32(0))), (best, scale)


def test_forced_pages_come_first_and_missing_ones_last(key):
    assert key.ordered(float("inf")) == FORCED and key.ordered(float("-inf")) == MISSING
    for scale in (1.0, float("nan"), float("inf"), -1e38):
        assert key.key(1, 1, 5, scale) == key.key(1, 0, 5, scale) == FORCED
        assert key.key(0, 0, 5, scale) == MISSING


def test_better_scores_have_larger_keys_and_equal_ones_the_same(key):
    values = np.sort(np.random.default_rng(2).normal(size=500).astype(np.float32))
    keys = [key.key(0, 1, 3, float(v)) for v in values]
    assert all(a < b for (a, b), (x, y) in zip(zip(keys, keys[1:]), zip(values, values[1:])) if np.float32(3) * x < np.float32(3) * y)
    assert key.key(0, 1, 0, 1.0) == key.key(0, 1, 0, -1.0)  # one zero
