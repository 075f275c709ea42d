"""Attention over prompts whose rows lie megabytes apart: offsets up to and beyond 31 and 32 bits (-m gpu)."""
import ctypes

import numpy as np
import pytest

from test_gpu_cache4 import BF16, F16, device, from_bits, to_bits
from test_gpu_prompt import Prompts

pytestmark = pytest.mark.gpu

STRIDE = 1 << 20  # elements from token to token: 2 MB


@pytest.mark.parametrize("kind,dim,queries,tokens,first", [
    (BF16, 64, 3, 831, 0),       # the longest sequence whose offsets the loads of whole pieces count
    (F16, 192, 40, 832, 0),      # and one more
    (BF16, 128, 5, 831, 1300),   # the sequence's first row lies beyond 31 bits
    (F16, 64, 70, 2130, 0)])     # its last ones beyond 32
def test_rows_far_apart(km, gpu, kind, dim, queries, tokens, first):
    rng = np.random.default_rng(dim)
    heads, group, rows = 2, 2, first + tokens
    s = Prompts(km, rng, heads, group, dim, [queries], [tokens], kind)
    held = km.DeviceBuffer(rows * STRIDE * 2)
    values_at = STRIDE // 2
    for t in range(tokens):
        for x, at in ((s.k, 0), (s.v, values_at)):
            bits = np.ascontiguousarray(to_bits(x[t], kind))
            km.check(km.hip_lib().kmx_h2d(ctypes.c_void_p(held.ptr.value + 2 * ((first + t) * STRIDE + at)), bits.ctypes.data, bits.nbytes))
            km.sync()
    q, out, lse = device(km, to_bits(s.q, kind)), device(km, np.zeros(s.q.shape, np.uint16)), device(km, np.zeros(s.q.shape[:3], np.float32))
    prompt = km.Prompt(1, heads * group, heads, dim, queries, rows, queries, tokens, device(km, np.int32([0, queries])), device(km, np.int32([first, rows])))
    for causal in (True, False):
        prompt.attend(kind, q, held, km.DeviceView(held.ptr.value + 2 * values_at, 0), out, s.scale, causal=causal, lse=lse, token_stride=STRIDE, head_stride=dim)
        km.sync()
        raw = out.read(np.uint16, s.q.size)
        got = from_bits(raw if kind == BF16 else raw.view(np.float16), kind).reshape(s.q.shape).astype(np.float64)
        want, want_lse, off, lse_off = s.expected(causal)
        assert np.all(np.abs(got - want) <= off), (np.abs(got - want) / off).max()
        assert np.all(np.abs(lse.read(np.float32, want_lse.size).reshape(want_lse.shape) - want_lse) <= lse_off)
    held.free()
