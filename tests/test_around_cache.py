"""What stands around the 4-bit cache without a GPU: structures, frequencies, and what the entry points refuse before any device work."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

from test_cache4 import DUMMY, batch_of, cache_of

ODD = ctypes.c_void_p((1 << 20) + 1)


def prompt_of(km, **other):
    fields = dict(sequences=2, query_heads=8, heads=4, dim=64, queries=20, tokens=30, max_queries=10, max_tokens=20, query_starts=DUMMY, token_starts=DUMMY)
    fields.update(other)
    return km.PromptStruct(*[fields[name] for name, _ in km.PromptStruct._fields_])


def rows_of(km, count=1, **other):
    fields = dict(in_=DUMMY, out=ctypes.c_void_p(1 << 24), in_token_stride=256, in_head_stride=64, out_token_stride=256, out_head_stride=64, heads=4)
    fields.update(other)
    one = km.RotaryRowsStruct(*[fields[name] for name, _ in km.RotaryRowsStruct._fields_])
    return (km.RotaryRowsStruct * count)(*[one] * count)


def test_structures_have_the_layout_of_the_header(km, tmp_path):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = tmp_path / "t.c"
    src.write_text('#include "kmx.h"\n#include <stdio.h>\n#include <stddef.h>\nint main(void){ printf("%zu %zu %zu %zu %zu %zu\\n", sizeof(kmx_rotary_rows), offsetof(kmx_rotary_rows, out_token_stride),'
                   ' offsetof(kmx_rotary_rows, heads), sizeof(kmx_prompt), offsetof(kmx_prompt, max_tokens), offsetof(kmx_prompt, token_starts)); return 0; }\n')
    subprocess.check_call(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(root, "include"), str(src), "-o", str(tmp_path / "t")])
    got = [int(v) for v in subprocess.check_output([str(tmp_path / "t")]).split()]
    r, p = km.RotaryRowsStruct, km.PromptStruct
    assert got == [ctypes.sizeof(r), r.out_token_stride.offset, r.heads.offset, ctypes.sizeof(p), p.max_tokens.offset, p.token_starts.offset]


@pytest.mark.parametrize("channels,base,stretch,length,slow,fast", [
    (128, 10000.0, 1.0, 0.0, 1.0, 32.0), (64, 500000.0, 8.0, 8192.0, 1.0, 4.0), (2, 10000.0, 4.0, 0.0, 0.0, 0.0), (96, 10000.0, 32.0, 4096.0, 1.0, 32.0),
    (128, 10000.0, 4.0, 2048.0, 2.0, 2.0), (6, 0.001, 1.0, 0.0, 1.0, 1.0)])
def test_frequencies(km, channels, base, stretch, length, slow, fast):
    """The first and last pair's frequency is known, those between by their definition; in 2^-64 of a turn, to the 53 bits that a double has of them."""
    got = km.rotary_turns(channels, base, stretch, length, slow, fast)
    i = np.arange(channels // 2)
    f = base ** (-2.0 * i / channels) / (2 * np.pi)
    share = np.zeros_like(f)
    if length:
        made = length * f
        share = np.where(made >= fast, 1.0, np.where(made <= slow, 0.0, (made - slow) / max(fast - slow, 1e-300)))
    want = f * (share + (1 - share) / stretch)
    assert np.all(np.abs(got.astype(np.float64) / 2.0 ** 64 - want % 1.0) <= 2.0 ** -50 * want + 2.0 ** -63)
    if length == 0 and stretch == 1:
        assert abs(float(got[0]) / 2.0 ** 64 - 1 / (2 * np.pi)) < 1e-16  # one radian a position
    if length and share[0] == 1 and share[-1] == 0:
        plain = km.rotary_turns(channels, base)
        # whole numbers on both sides: half a unit off each, that of the stretched one times the stretch, and the 53 bits of the doubles that they come from
        assert got[0] == plain[0] and abs(float(got[-1]) * stretch - float(plain[-1])) <= 0.5 * stretch + 0.5 + 2.0 ** -50 * float(plain[-1])


@pytest.mark.parametrize("bad", [(3, 1e4, 1, 0, 1, 32), (4, 0, 1, 0, 1, 32), (4, -1, 1, 0, 1, 32), (4, np.nan, 1, 0, 1, 32), (4, np.inf, 1, 0, 1, 32), (4, 1e4, 0, 0, 1, 32), (4, 1e4, np.nan, 0, 1, 32),
                                 (4, 1e4, 1, -1, 1, 32), (4, 1e4, 1, np.inf, 1, 32), (4, 1e4, 1, 8, 2, 1), (4, 1e4, 1, 8, np.nan, 1), (4, 1e4, 1, 8, -1, 1)])
def test_frequencies_that_are_refused(km, bad):
    with pytest.raises(km.KmxError) as e:
        km.rotary_turns(*bad)
    assert e.value.code == km.KMX_ERR_INVALID_ARGUMENT
    assert km.hip_lib().kmx_rotary_turns(4, 1e4, 1, 0, 1, 32, None) == km.KMX_ERR_INVALID_ARGUMENT
    assert km.rotary_turns(0).shape == (0,)


def test_rotations_that_are_refused(km):
    lib = km.hip_lib()
    invalid, unsupported = km.KMX_ERR_INVALID_ARGUMENT, km.KMX_ERR_UNSUPPORTED

    def call(code, word, kind=km.TYPE_BF16, rows=None, sets=1, tokens=5, dim=64, channels=32, turns=DUMMY, positions=DUMMY, halves=1, inverse=0, gain=1.0):
        rc = lib.kmx_rotary(kind, rows_of(km) if rows is None else rows, sets, tokens, dim, channels, turns, positions, halves, inverse, gain)
        assert rc == code and word in lib.kmx_last_error(), (rc, lib.kmx_last_error())

    call(invalid, b"type 7", kind=7)
    call(invalid, b"33 rotated", channels=33)
    call(invalid, b"66 rotated", channels=66)
    call(invalid, b"0 or 1", halves=2)
    call(invalid, b"0 or 1", inverse=-1)
    call(invalid, b"gain", gain=float("nan"))
    call(unsupported, b"5 sets", rows=rows_of(km, 5), sets=5)
    call(invalid, b"null device", rows=rows_of(km, in_=None))
    call(invalid, b"null device", rows=rows_of(km, out=None))
    call(invalid, b"element", rows=rows_of(km, in_=ODD))
    call(invalid, b"element", kind=km.TYPE_F32, rows=rows_of(km, out=ctypes.c_void_p((1 << 20) + 2)))
    call(invalid, b"head stride", rows=rows_of(km, out_head_stride=63))
    call(invalid, b"token stride", rows=rows_of(km, out_token_stride=63))
    call(invalid, b"one set of strides", rows=rows_of(km, out=DUMMY, out_token_stride=512))
    call(invalid, b"one set of strides", rows=rows_of(km, out=DUMMY, out_head_stride=128))
    call(unsupported, b"too many heads", rows=rows_of(km, heads=1 << 25))
    call(invalid, b"null positions", positions=None)
    call(invalid, b"null positions", turns=None)
    assert lib.kmx_rotary(km.TYPE_BF16, None, 1, 5, 64, 32, DUMMY, DUMMY, 1, 0, 1.0) == invalid
    for nothing in (dict(tokens=0), dict(sets=0), dict(dim=0, channels=0), dict(rows=rows_of(km, heads=0)), dict(channels=0, rows=rows_of(km, out=DUMMY))):
        call(km.KMX_OK, b"", **nothing)


def test_prompts_that_are_refused(km):
    lib = km.hip_lib()
    invalid, unsupported = km.KMX_ERR_INVALID_ARGUMENT, km.KMX_ERR_UNSUPPORTED

    def call(code, word, kind=km.TYPE_BF16, q=DUMMY, k=DUMMY, v=DUMMY, out=DUMMY, ots=512, ohs=64, scale=1.0, causal=1, prompt=True, **other):
        rc = lib.kmx_prompt_attend(prompt_of(km, **other) if prompt else None, kind, q, 512, 64, k, v, 256, 64, out, ots, ohs, None, scale, causal)
        assert rc == code and word in lib.kmx_last_error(), (rc, lib.kmx_last_error())

    call(invalid, b"null prompt", prompt=False)
    call(invalid, b"no multiple", query_heads=6)
    call(invalid, b"no multiple", heads=0)
    call(invalid, b"no multiple", query_heads=0)
    for dim in (0, 48, 288):
        call(unsupported, b"dim %d" % dim, dim=dim)
    call(unsupported, b"F16 or KMX_BF16", kind=km.TYPE_F32)
    call(invalid, b"type 3", kind=3)
    call(invalid, b"causal", causal=2)
    call(invalid, b"scale", scale=float("inf"))
    call(invalid, b"scale", scale=float("nan"))
    call(invalid, b"null device", query_starts=None)
    call(invalid, b"null device", token_starts=None)
    call(unsupported, b"31 bits", queries=1 << 31)
    call(unsupported, b"31 bits", tokens=1 << 31)
    for name in "qkv":
        call(invalid, b"null device", **{name: None})
        call(invalid, b"2 bytes", **{name: ODD})
    call(invalid, b"null device", out=None)
    call(invalid, b"head stride", ohs=63)
    call(invalid, b"token stride", ots=63)
    for nothing in (dict(sequences=0), dict(queries=0), dict(max_queries=0)):
        call(km.KMX_OK, b"", q=None, k=None, v=None, out=None, query_starts=None, token_starts=None, **nothing)
    assert lib.kmx_prompt_reserve(48) == lib.kmx_prompt_reserve(0) == lib.kmx_prompt_reserve(288) == unsupported and b"multiple of 32" in lib.kmx_last_error()


def test_shared_prefixes_that_are_refused(km):
    lib, c = km.hip_lib(), cache_of(km)
    invalid, unsupported = km.KMX_ERR_INVALID_ARGUMENT, km.KMX_ERR_UNSUPPORTED

    def call(code, word, c=c, prefix=None, batch=None, kind=km.TYPE_BF16, q=DUMMY, out=DUMMY, ots=512, ohs=64, scale=1.0, causal=1):
        rc = lib.kmx_cache4_attend_shared(c, batch_of(km, sequences=1) if prefix is None else prefix or None, batch_of(km) if batch is None else batch or None, kind, q, 512, 64, out, ots, ohs, None, scale, causal)
        assert rc == code and word in lib.kmx_last_error(), (rc, lib.kmx_last_error())

    call(invalid, b"heads", c=cache_of(km, heads=0))
    call(invalid, b"null batch", prefix=0)
    call(invalid, b"null batch", batch=0)
    call(invalid, b"prefixes have 3 rows", prefix=batch_of(km, tokens=3))
    call(invalid, b"prefixes have 2 rows of 4", prefix=batch_of(km, query_heads=4))
    call(invalid, b"no multiple", batch=batch_of(km, query_heads=6))
    call(invalid, b"null device", prefix=batch_of(km, table=None))
    call(invalid, b"null device", batch=batch_of(km, lengths=None))
    call(unsupported, b"31 bits", prefix=batch_of(km, max_length=1 << 31))
    call(unsupported, b"F16 or KMX_BF16", kind=km.TYPE_F32)
    call(invalid, b"causal", causal=3)
    call(invalid, b"scale", scale=float("nan"))
    call(invalid, b"null device", q=None)
    call(invalid, b"2 bytes", out=ODD)
    call(invalid, b"head stride", ohs=63)
    call(invalid, b"token stride", ots=63)
    call(km.KMX_OK, b"", batch=batch_of(km, sequences=0, starts=None), q=None)
    for bad in ((None, batch_of(km)), (batch_of(km), None), (batch_of(km, tokens=3), batch_of(km)), (batch_of(km, query_heads=6), batch_of(km, query_heads=6))):
        assert lib.kmx_cache4_reserve_shared(c, *bad) == invalid


def test_weighing_and_eviction_that_are_refused(km):
    lib, c = km.hip_lib(), cache_of(km)
    invalid, unsupported = km.KMX_ERR_INVALID_ARGUMENT, km.KMX_ERR_UNSUPPORTED

    def weigh(code, word, c=c, b=None, kind=km.TYPE_F16, q=DUMMY, lse=DUMMY, scale=1.0, causal=1, weights=DUMMY):
        rc = lib.kmx_cache4_weigh(c, batch_of(km) if b is None else b or None, kind, q, 512, 64, lse, scale, causal, weights)
        assert rc == code and word in lib.kmx_last_error(), (rc, lib.kmx_last_error())

    weigh(invalid, b"null device", c=cache_of(km, blocks=None))
    weigh(invalid, b"null batch", b=0)
    weigh(invalid, b"no multiple", b=batch_of(km, query_heads=6))
    weigh(unsupported, b"F16 or KMX_BF16", kind=km.TYPE_F32)
    weigh(invalid, b"scale", scale=float("inf"))
    weigh(invalid, b"causal", causal=2)
    weigh(invalid, b"null device", q=None)
    weigh(invalid, b"null device", lse=None)
    weigh(invalid, b"null device", weights=None)
    weigh(invalid, b"element", weights=ctypes.c_void_p((1 << 20) + 2))
    weigh(unsupported, b"too many", b=batch_of(km, sequences=70000))
    weigh(unsupported, b"31 bits", b=batch_of(km, tokens=1 << 31, max_queries=1 << 31))
    for nothing in (dict(sequences=0), dict(tokens=0), dict(max_queries=0), dict(max_length=0), dict(table_stride=0)):
        weigh(km.KMX_OK, b"", b=batch_of(km, **nothing), q=None)

    def evict(code, word, c=c, b=None, weights=DUMMY, keep=10, first=2, recent=3, kept=DUMMY, left=ctypes.c_void_p(1 << 24)):
        rc = lib.kmx_cache4_evict(c, batch_of(km) if b is None else b or None, weights, keep, first, recent, kept, left)
        assert rc == code and word in lib.kmx_last_error(), (rc, lib.kmx_last_error())

    evict(unsupported, b"dim 48", c=cache_of(km, dim=48))
    evict(invalid, b"null batch", b=0)
    evict(invalid, b"10 tokens have no room", first=8)
    evict(invalid, b"no room", keep=0xFFFFFFFF, first=0xFFFFFFFF, recent=1)
    evict(unsupported, b"262144", b=batch_of(km, max_length=262145))
    evict(invalid, b"null device", b=batch_of(km, lengths=None))
    evict(invalid, b"null device", b=batch_of(km, table=None))
    evict(invalid, b"null device", weights=None)
    evict(invalid, b"null device", kept=None)
    evict(invalid, b"null device", left=None)
    evict(invalid, b"two arrays", left=DUMMY)
    evict(invalid, b"element", kept=ctypes.c_void_p((1 << 20) + 2))
    evict(unsupported, b"too many", b=batch_of(km, sequences=70000))
    evict(km.KMX_OK, b"", b=batch_of(km, sequences=0, lengths=None, table=None), weights=None, kept=None, left=None)


def test_prompts_are_shared_out_whole_and_within_the_reserved_room(tmp_path):
    """Launch shapes of the attention over prompts (csrc/prompt_plan.h): every tile in one part, none of the longest sequence's parts empty, room as kmx_prompt_reserve makes it."""
    source = tmp_path / "plan.cpp"
    source.write_text(r"""
#include "prompt_plan.h"
#include <initializer_list>
#include <cstdio>
using namespace kmx;
int main()
{
	unsigned parts = 0;
	for (uint32_t J = 1; J <= 8; ++J)
		for (uint32_t heads : { 1u, 3u, 8u, 64u })
			for (uint32_t group : { 1u, 4u, 7u })
				for (uint32_t sequences : { 1u, 5u, 300u })
					for (uint32_t queries : { 1u, 31u, 500u, 8192u, 0x7FFFFFFFu })
						for (uint32_t tokens : { 0u, 1u, 33u, 64u, 129u, 1000u, 8192u, 100001u, 0x7FFFFFFFu }) {
							const PromptPlan p = plan_prompt(PromptShape{ J, heads, group, sequences, queries, tokens, 256 });
							const uint64_t rows = (uint64_t)queries * group, tile = p.wide ? 256 : 128, tiles = ((uint64_t)tokens + 31) / 32;
							const uint64_t units = (rows + tile - 1) / tile * heads * sequences;
							if (p.units == 0) {
								if (rows <= 0x7FFFFF00u && units <= 0x7FFFFFFFu) return printf("refused %u %u %u %u %u\n", J, heads, group, sequences, queries), 1;
								continue;
							}
							if (p.units != units || (uint64_t)p.units * p.parts > 0x7FFFFFFFu || (p.wide ? J < 3 || J > 6 : J == 5 || J == 6)) return printf("units\n"), 1;
							if ((uint64_t)p.parts * p.tiles_per_part < tiles || p.parts == 0 || (p.parts > 1 && (uint64_t)(p.parts - 1) * p.tiles_per_part >= tiles)) return printf("parts\n"), 1;
							if (p.parts > 1 && p.tiles_per_part < PROMPT_LEAST) return printf("short parts\n"), 1;
							if (prompt_floats(p, J) > most_prompt_floats(J, 256) || 4 * prompt_floats(p, J) > (64u << 20)) return printf("room\n"), 1;
							parts += p.parts > 1;
						}
	printf("%u", parts);
	return parts < 100;
}
""")
    import os
    import subprocess
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cuda-kmeans_amd", "csrc")
    program = tmp_path / "plan"
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", csrc, str(source), "-o", str(program)], check=True)
    ran = subprocess.run([str(program)], capture_output=True, text=True)
    assert ran.returncode == 0, ran.stdout
