"""CPU: the cache's C entries refuse bad arguments before anything touches a device."""
import ctypes

import pytest

from int4matmul_kernels_b200 import capi


def cache(**changes):
    c = dict(k=16, v=16, scales=16, pages=4, heads=2, page_size=16, head_dim=128, k_page_stride=4096, k_head_stride=2048, k_token_stride=128,
             v_page_stride=4096, v_head_stride=2048, v_token_stride=128, type=capi.CACHE_INT8)
    c.update(changes)
    return ctypes.byref(capi.Cache(*(c[n] for n, _ in capi.Cache._fields_)))


BAD_CACHES = [(dict(type=2), capi.ERR_UNSUPPORTED), (dict(head_dim=96), capi.ERR_UNSUPPORTED), (dict(page_size=24), capi.ERR_UNSUPPORTED),
              (dict(pages=0), capi.ERR_SHAPE), (dict(heads=0), capi.ERR_SHAPE), (dict(pages=1 << 31), capi.ERR_SHAPE), (dict(k=None), capi.ERR_NULL),
              (dict(scales=None), capi.ERR_NULL), (dict(v=8), capi.ERR_ALIGN), (dict(scales=4), capi.ERR_ALIGN), (dict(k_token_stride=72), capi.ERR_ALIGN),
              (dict(v_page_stride=4097), capi.ERR_ALIGN)]


@pytest.mark.parametrize("changes,status", BAD_CACHES)
def test_caches(built_library, changes, status):
    lib = built_library
    assert lib.i4mm_cache_write(cache(**changes), 16, 16, 0, 1, 128, 128, 128, 128, 16, None) == status
    assert lib.i4mm_cache_read(cache(**changes), 16, 16, 0, 1, 16, None) == status
    assert lib.i4mm_cache_attention(cache(**changes), 16, 16, 0, 1, 2, 256, 128, 16, 1, 1, 16, None, 1, 1, 1.0, 0, 16, 1 << 30, None) == status


def test_null_cache(built_library):
    assert built_library.i4mm_cache_read(None, 16, 16, 0, 1, 16, None) == capi.ERR_NULL


def test_write_and_read(built_library):
    def write(k=16, v=16, type=0, tokens=1, strides=(128, 128, 128, 128), slots=16):
        return built_library.i4mm_cache_write(cache(), k, v, type, tokens, *strides, slots, None)
    assert write(tokens=0) == capi.OK
    assert write(type=2) == capi.ERR_UNSUPPORTED
    assert write(tokens=-1) == capi.ERR_SHAPE
    assert write(k=None) == capi.ERR_NULL and write(slots=None) == capi.ERR_NULL
    assert write(v=8) == capi.ERR_ALIGN and write(strides=(128, 4, 128, 128)) == capi.ERR_ALIGN
    read = lambda **a: built_library.i4mm_cache_read(cache(), a.get("k", 16), a.get("v", 16), a.get("type", 0), a.get("tokens", 1), a.get("slots", 16), None)  # noqa: E731
    assert read(tokens=0) == capi.OK and read(tokens=-1) == capi.ERR_SHAPE
    assert read(type=7) == capi.ERR_UNSUPPORTED and read(v=None) == capi.ERR_NULL and read(k=8) == capi.ERR_ALIGN


def test_plan(built_library):
    def plan(n=1, seq=16, new=16, table=16, width=1, stride=1, free=16, capacity=1, count=16, page=16, tokens=1, outs=(16,) * 6):
        return built_library.i4mm_cache_plan(n, seq, new, table, width, stride, free, capacity, count, page, tokens, *outs, None)
    assert plan(page=20) == capi.ERR_UNSUPPORTED
    assert plan(n=-1) == capi.ERR_SHAPE and plan(n=16385) == capi.ERR_SHAPE and plan(width=2) == capi.ERR_SHAPE and plan(tokens=-1) == capi.ERR_SHAPE
    assert plan(capacity=-1) == capi.ERR_SHAPE
    assert plan(seq=None) == capi.ERR_NULL and plan(table=None) == capi.ERR_NULL and plan(free=None) == capi.ERR_NULL and plan(count=None) == capi.ERR_NULL
    for i in range(6):
        assert plan(outs=(16,) * i + (None,) + (16,) * (5 - i)) == capi.ERR_NULL
        assert plan(outs=(16,) * i + (18,) + (16,) * (5 - i)) == capi.ERR_ALIGN


def test_attention(built_library):
    def attend(out=16, q=16, type=0, tokens=1, heads=2, strides=(256, 128), table=16, width=1, stride=1, seq=16, cu=None, n=1, longest=1, window=0, ws=16,
               size=1 << 30):
        return built_library.i4mm_cache_attention(cache(), out, q, type, tokens, heads, *strides, table, width, stride, seq, cu, n, longest, 1.0, window,
                                                  ws, size, None)
    assert attend(tokens=0, n=0) == capi.OK
    assert attend(type=3) == capi.ERR_UNSUPPORTED
    for bad in (dict(heads=3), dict(heads=0), dict(tokens=-1), dict(tokens=1 << 31), dict(n=2), dict(n=-1), dict(n=16385, cu=16), dict(width=2), dict(longest=-1),
                dict(window=-1), dict(width=1 << 28, stride=1 << 28)):
        assert attend(**bad) == capi.ERR_SHAPE, bad
    for bad in (dict(out=None), dict(q=None), dict(seq=None), dict(table=None)):
        assert attend(**bad) == capi.ERR_NULL, bad
    for bad in (dict(out=8), dict(q=8), dict(table=18), dict(cu=17), dict(strides=(256, 4)), dict(ws=24)):
        assert attend(**bad) == capi.ERR_ALIGN, bad
    assert attend(ws=None) == capi.ERR_WORKSPACE and attend(size=8) == capi.ERR_WORKSPACE
