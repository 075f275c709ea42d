"""Rotation of so many rows that a lane takes eight heads of a token, the most there are (csrc/rotary.hip), of several sets (-m gpu)."""
import numpy as np
import pytest

from test_gpu_cache4 import BF16, F16, F32
from test_gpu_rotary import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,dim,channels,tokens,how", [(F16, 24, 16, 20001, dict(gaps=(1, 0), out_gaps=(0, 3), offset=1, halves=False)), (BF16, 24, 24, 20001, dict(gaps=(1, 2))),
                                                           (F32, 8, 8, 240001, {}), (F32, 8, 8, 240001, dict(in_place=True, inverse=True))])
def test_eight_heads_a_lane(km, gpu, kind, dim, channels, tokens, how):
    """tokens x 9 heads x pieces of a row (16 bytes and their partners, or a pair of channels) are more than eight times the 1024 x 256 lanes that fill the chip; nine heads: eight and one."""
    vec = kind == F32
    pieces = channels // 2 // (4 if vec else 1) + (dim - channels) // 2
    assert tokens * 9 * pieces >= 8 * 256 * 1024
    check(km, np.random.default_rng(dim), kind, tokens, (6, 1, 2), dim, channels, **how)
