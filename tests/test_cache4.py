"""The 4-bit cache without a GPU: its structures, sizes and rounded levels, and what its entry points refuse before any device work."""
import ctypes

import numpy as np
import pytest

DUMMY = ctypes.c_void_p(1 << 20)  # an address that no refused call follows


def cache_of(km, **other):
    fields = dict(blocks=DUMMY, bounds=DUMMY, levels=DUMMY, heads=4, dim=64, page_tokens=32, page_count=10)
    fields.update(other)
    return km.Cache4Struct(*[fields[name] for name, _ in km.Cache4Struct._fields_])


def batch_of(km, **other):
    fields = dict(sequences=2, query_heads=8, tokens=2, max_queries=1, max_length=100, table_stride=4, starts=DUMMY, lengths=DUMMY, table=DUMMY)
    fields.update(other)
    return km.Cache4BatchStruct(*[fields[name] for name, _ in km.Cache4BatchStruct._fields_])


def test_structures_have_the_layout_of_the_header(km, tmp_path):
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = tmp_path / "t.c"
    src.write_text('#include "kmx.h"\n#include <stdio.h>\n#include <stddef.h>\nint main(void){ printf("%zu %zu %zu %zu %zu %zu %d %d %d\\n", sizeof(kmx_cache4), offsetof(kmx_cache4, heads),'
                   ' offsetof(kmx_cache4, page_count), sizeof(kmx_cache4_batch), offsetof(kmx_cache4_batch, starts), offsetof(kmx_cache4_batch, table), KMX_F32, KMX_F16, KMX_BF16); return 0; }\n')
    subprocess.check_call(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(root, "include"), str(src), "-o", str(tmp_path / "t")])
    got = [int(v) for v in subprocess.check_output([str(tmp_path / "t")]).split()]
    c, b = km.Cache4Struct, km.Cache4BatchStruct
    assert got == [ctypes.sizeof(c), c.heads.offset, c.page_count.offset, ctypes.sizeof(b), b.starts.offset, b.table.offset, km.TYPE_F32, km.TYPE_F16, km.TYPE_BF16]


@pytest.mark.parametrize("heads,dim,page,pages", [(1, 32, 16, 0), (1, 32, 16, 1), (8, 128, 64, 1000), (5, 96, 256, 7), (64, 256, 128, 60000)])
def test_sizes(km, heads, dim, page, pages):
    # a token of a head: two codes of 4 bits a channel and two halves for each 32; a bound: two bytes a channel and a float
    assert km.Cache4.sizes(heads, dim, page, pages) == (pages * page * heads * (dim + 2 * 2 * dim // 32), pages * heads * (2 * dim + 4))


def test_levels_are_rounded_to_six_bits(km):
    rng = np.random.default_rng(3)
    sets = np.sort(rng.random((50, 8), dtype=np.float32), axis=1)
    sets[0] = [0, 2.0 ** -24, 2.0 ** -20, 2.0 ** -15, 2.0 ** -14, 0.5, 65 / 128, 1]
    got = km.cache4_round_levels(sets).astype(np.float64)
    part, power = np.frexp(sets.astype(np.float64))
    want = np.ldexp(np.round(part * 64) / 64, power)  # ties to the even one
    fine = power > -14                                  # below, half precision has fewer places
    assert np.array_equal(got[fine], want[fine])
    assert np.abs(got - sets).max() <= 2.0 ** -7 and np.all(np.abs(got - sets)[~fine] <= 2.0 ** -20)
    assert np.all(np.diff(got, axis=1) >= 0) and got.max() <= 1
    assert got[0, 6] == 0.5  # 65/128 has seven bits: the even one
    assert km.cache4_round_levels(np.zeros((0, 8))).shape == (0, 8)


@pytest.mark.parametrize("bad", [[0, .1, .2, .3, .4, .5, .6, 1.5], [-.1, .1, .2, .3, .4, .5, .6, .7], [0, .2, .1, .3, .4, .5, .6, .7], [0, .1, .2, .3, np.nan, .5, .6, .7]])
def test_levels_that_are_refused(km, bad):
    with pytest.raises(km.KmxError) as e:
        km.cache4_round_levels(np.float32(bad))
    assert e.value.code == km.KMX_ERR_INVALID_ARGUMENT
    with pytest.raises(ValueError):
        km.cache4_round_levels(np.zeros(7))


@pytest.mark.parametrize("other,code,word", [
    (dict(heads=0), 1, b"heads"), (dict(dim=0), 2, b"dim 0"), (dict(dim=48), 2, b"dim 48"), (dict(dim=288), 2, b"dim 288"),
    (dict(page_tokens=8), 2, b"pages of 8"), (dict(page_tokens=48), 2, b"pages of 48"), (dict(page_tokens=512), 2, b"pages of 512"),
    (dict(page_count=1 << 27), 2, b"31 bits"), (dict(blocks=None), 1, b"null"), (dict(levels=None), 1, b"null"),
    (dict(blocks=ctypes.c_void_p((1 << 20) + 8)), 1, b"16 bytes")])
def test_caches_that_are_refused(km, other, code, word):
    lib, c, b = km.hip_lib(), cache_of(km, **other), batch_of(km)
    for call in (lambda: lib.kmx_cache4_write(c, km.TYPE_BF16, DUMMY, DUMMY, 256, 64, DUMMY, 3), lambda: lib.kmx_cache4_read(c, km.TYPE_BF16, DUMMY, DUMMY, 256, 64, DUMMY, 3),
                 lambda: lib.kmx_cache4_bound(c, DUMMY, DUMMY, 3), lambda: lib.kmx_cache4_select(c, b, km.TYPE_BF16, DUMMY, 512, 64, DUMMY, 4, 1, 1, 1),
                 lambda: lib.kmx_cache4_attend(c, b, km.TYPE_BF16, DUMMY, 512, 64, DUMMY, 512, 64, None, 1.0, 1, None, 0)):
        assert call() == code and word in lib.kmx_last_error(), lib.kmx_last_error()


def test_arguments_that_are_refused(km):
    lib, c, b = km.hip_lib(), cache_of(km), batch_of(km)
    invalid, unsupported = km.KMX_ERR_INVALID_ARGUMENT, km.KMX_ERR_UNSUPPORTED

    def refused(rc, code, word):
        assert rc == code and word in lib.kmx_last_error(), (rc, lib.kmx_last_error())

    refused(lib.kmx_cache4_sizes(None, None, None), invalid, b"null cache")
    refused(lib.kmx_cache4_write(c, 7, DUMMY, DUMMY, 256, 64, DUMMY, 3), invalid, b"type 7")
    refused(lib.kmx_cache4_write(c, km.TYPE_F32, None, DUMMY, 256, 64, DUMMY, 3), invalid, b"null device")
    refused(lib.kmx_cache4_write(c, km.TYPE_F32, ctypes.c_void_p((1 << 20) + 2), DUMMY, 256, 64, DUMMY, 3), invalid, b"element")
    refused(lib.kmx_cache4_read(c, km.TYPE_F32, DUMMY, DUMMY, 63, 64, DUMMY, 3), invalid, b"token stride")
    refused(lib.kmx_cache4_read(c, km.TYPE_F32, DUMMY, DUMMY, 256, 63, DUMMY, 3), invalid, b"head stride")
    refused(lib.kmx_cache4_read(c, km.TYPE_F32, DUMMY, DUMMY, 256, 64, None, 3), invalid, b"null device")
    refused(lib.kmx_cache4_bound(cache_of(km, bounds=None), DUMMY, DUMMY, 3), invalid, b"no bounds")
    refused(lib.kmx_cache4_bound(c, DUMMY, None, 3), invalid, b"null device")
    select = lambda c=c, b=b, t=km.TYPE_BF16, q=DUMMY, out=DUMMY, top=4, first=1, last=1, causal=1: lib.kmx_cache4_select(c, b, t, q, 512, 64, out, top, first, last, causal)  # noqa: E731
    refused(select(c=cache_of(km, bounds=None)), invalid, b"no bounds")
    refused(select(t=km.TYPE_F32), unsupported, b"F16 or KMX_BF16")
    refused(select(top=0), invalid, b"top 0")
    refused(select(top=3, first=2, last=2), invalid, b"top 3")
    refused(select(q=None), invalid, b"null device")
    refused(select(out=None), invalid, b"null device")
    refused(select(causal=2), invalid, b"causal")
    refused(select(b=None), invalid, b"null batch")
    attend = lambda c=c, b=b, t=km.TYPE_BF16, q=DUMMY, out=DUMMY, ots=512, ohs=64, scale=1.0, causal=1, chosen=None, top=0: lib.kmx_cache4_attend(  # noqa: E731
        c, b, t, q, 512, 64, out, ots, ohs, None, scale, causal, chosen, top)
    refused(attend(b=None), invalid, b"null batch")
    refused(attend(b=batch_of(km, query_heads=6)), invalid, b"no multiple")
    refused(attend(b=batch_of(km, query_heads=0)), invalid, b"no multiple")
    refused(attend(b=batch_of(km, starts=None)), invalid, b"null device")
    refused(attend(b=batch_of(km, table=None)), invalid, b"null device")
    refused(attend(b=batch_of(km, max_length=1 << 31)), unsupported, b"31 bits")
    refused(attend(t=km.TYPE_F32), unsupported, b"F16 or KMX_BF16")
    refused(attend(t=3), invalid, b"type 3")
    refused(attend(scale=float("nan")), invalid, b"scale")
    refused(attend(scale=float("inf")), invalid, b"scale")
    refused(attend(chosen=DUMMY), invalid, b"top is 0")
    refused(attend(q=None), invalid, b"null device")
    refused(attend(out=ctypes.c_void_p((1 << 20) + 1)), invalid, b"2 bytes")
    refused(attend(ohs=63), invalid, b"head stride")
    refused(attend(ots=63), invalid, b"token stride")
    refused(lib.kmx_cache4_reserve(c, batch_of(km, query_heads=6), 0), invalid, b"no multiple")
    refused(lib.kmx_cache4_reserve(c, None, 0), invalid, b"null batch")


def test_calls_with_nothing_to_do_need_no_device(km):
    lib, c = km.hip_lib(), cache_of(km)
    assert lib.kmx_cache4_write(c, km.TYPE_F32, None, None, 256, 64, None, 0) == km.KMX_OK
    assert lib.kmx_cache4_read(c, km.TYPE_F32, None, None, 256, 64, None, 0) == km.KMX_OK
    assert lib.kmx_cache4_bound(c, None, None, 0) == km.KMX_OK
    for nothing in (dict(sequences=0), dict(tokens=0), dict(max_queries=0)):
        b = batch_of(km, starts=None, lengths=None, table=None, **nothing)
        assert lib.kmx_cache4_select(c, b, km.TYPE_F16, None, 512, 64, None, 4, 1, 1, 1) == km.KMX_OK
        assert lib.kmx_cache4_attend(c, b, km.TYPE_F16, None, 512, 64, None, 512, 64, None, 1.0, 1, None, 0) == km.KMX_OK
    assert lib.kmx_last_error() == b""
