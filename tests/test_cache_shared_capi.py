"""CPU: the C entries of positions, head norms and shared prefixes refuse bad arguments before anything touches a device."""
import pytest

from int4matmul_kernels_b200 import capi
from test_cache_capi import BAD_CACHES, cache


def test_angles(built_library):
    def angles(out=16, positions=16, freqs=16, tokens=1, pairs=8):
        return built_library.i4mm_cache_angles(out, positions, freqs, tokens, pairs, None)
    assert angles(tokens=0) == capi.OK and angles(pairs=0) == capi.OK
    for bad in (dict(tokens=-1), dict(tokens=1 << 31), dict(pairs=-8), dict(pairs=136)):
        assert angles(**bad) == capi.ERR_SHAPE, bad
    assert angles(pairs=12) == capi.ERR_UNSUPPORTED
    for name in ("out", "positions", "freqs"):
        assert angles(**{name: None}) == capi.ERR_NULL
    for bad in (dict(out=8), dict(positions=18), dict(freqs=4)):
        assert angles(**bad) == capi.ERR_ALIGN, bad


def test_share(built_library):
    def share(n=1, of=16, seq=16, cu=16, tokens=1, outs=(16,) * 4):
        return built_library.i4mm_cache_share(n, of, seq, cu, tokens, *outs, None)
    for bad in (dict(n=-1), dict(n=16385), dict(tokens=-1), dict(tokens=(1 << 30) + 1)):
        assert share(**bad) == capi.ERR_SHAPE, bad
    for name in ("of", "seq", "cu"):
        assert share(**{name: None}) == capi.ERR_NULL and share(**{name: 18}) == capi.ERR_ALIGN
    for i in range(4):
        assert share(outs=(16,) * i + (None,) + (16,) * (3 - i)) == capi.ERR_NULL
        assert share(outs=(16,) * i + (18,) + (16,) * (3 - i)) == capi.ERR_ALIGN


@pytest.mark.parametrize("changes,status", BAD_CACHES)
def test_caches(built_library, changes, status):
    lib, bad = built_library, cache(**changes)
    assert lib.i4mm_cache_append(bad, 16, 16, 16, 16, 0, 1, 2, 256, 128, 256, 128, 256, 128, 16, 16, 8, 0, None, None, 1e-6, None) == status
    assert lib.i4mm_cache_attention_shared(bad, 16, 16, 0, 1, 2, 256, 128, 16, 1, 1, 16, None, 1, 1, 1.0, 0, 16, 16, 16, 1, 16, 1 << 30, 16, 1 << 30,
                                           None) == status


def test_append(built_library):
    def append(out=16, q=16, k=16, v=16, type=0, tokens=1, heads=2, strides=(256, 128) * 3, slots=16, angles=16, pairs=64, beside=0, qw=None, kw=None):
        return built_library.i4mm_cache_append(cache(), out, q, k, v, type, tokens, heads, *strides, slots, angles, pairs, beside, qw, kw, 1e-6, None)
    assert append(tokens=0) == capi.OK
    assert append(type=2) == capi.ERR_UNSUPPORTED and append(pairs=12) == capi.ERR_UNSUPPORTED
    for bad in (dict(tokens=-1), dict(heads=0), dict(heads=65536), dict(tokens=1 << 31), dict(pairs=72), dict(pairs=-8)):
        assert append(**bad) == capi.ERR_SHAPE, bad
    for name in ("out", "q", "k", "v", "slots", "angles"):
        assert append(**{name: None}) == capi.ERR_NULL, name
    for bad in (dict(out=8), dict(q=8), dict(k=24), dict(v=8), dict(slots=18), dict(angles=8), dict(qw=8), dict(kw=4), dict(strides=(256, 4) + (256, 128) * 2)):
        assert append(**bad) == capi.ERR_ALIGN, bad


def test_attention(built_library):
    lib = built_library
    enough = lib.i4mm_cache_shared_scratch_bytes(1, 2, 128)
    assert enough == 16 + 2 * 128 * 4
    assert lib.i4mm_cache_shared_scratch_bytes(3, 1, 64) == 32 + 3 * 64 * 4
    assert lib.i4mm_cache_shared_scratch_bytes(-1, 2, 128) == 0

    def attend(tokens=1, of=16, starts=16, rows=16, listed=1, scratch=16, size=enough, ws=16, ws_size=1 << 30, heads=2):
        return lib.i4mm_cache_attention_shared(cache(), 16, 16, 0, tokens, heads, 256, 128, 16, 1, 1, 16, None, min(tokens, 1), 1, 1.0, 0, of, starts, rows, listed,
                                               scratch, size, ws, ws_size, None)
    assert attend(tokens=0) == capi.OK
    assert attend(listed=0) == capi.ERR_SHAPE and attend(heads=3) == capi.ERR_SHAPE and attend(listed=1 << 31) == capi.ERR_SHAPE
    for name in ("of", "starts", "rows", "scratch"):
        assert attend(**{name: None}) == capi.ERR_NULL, name
    for bad in (dict(of=18), dict(starts=18), dict(rows=18), dict(scratch=24), dict(ws=24)):
        assert attend(**bad) == capi.ERR_ALIGN, bad
    assert attend(size=enough - 1) == capi.ERR_WORKSPACE and attend(ws=None) == capi.ERR_WORKSPACE and attend(ws_size=8) == capi.ERR_WORKSPACE
    assert lib.i4mm_last_attention_kernels() == 0


def test_attention_counts_in_32_bits(built_library):
    """A table and rows of which there could be more than 2^31 tiles are refused; half of that is not what is wrong."""
    lib, wide = built_library, ((1 << 31) - 1 - 127) // 16

    def attend(tokens, size):
        return lib.i4mm_cache_attention_shared(cache(), 16, 16, 0, tokens, 2, 256, 128, 16, wide, wide, 16, 16, 1, 1, 1.0, 0, 16, 16, 16, tokens, 16, size, 16, 1 << 30, None)
    # 2 key heads, 2^24 + 1 tiles of 128 tokens: 63 tiles of 64 rows are counted, 64 are not
    tokens = 64 * 63
    assert attend(tokens, lib.i4mm_cache_shared_scratch_bytes(tokens, 2, 128)) == capi.ERR_TOO_LARGE
    assert attend(tokens, 16) == capi.ERR_WORKSPACE and lib.i4mm_last_attention_kernels() == 0
