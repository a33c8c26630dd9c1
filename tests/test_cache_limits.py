"""CPU: sizes whose loops would pass 32 bits are refused before anything touches a device, and strides that mean nothing are not."""
import ctypes

import pytest
import torch

from int4matmul_kernels_b200 import capi


def test_tables_of_a_step_of_2_to_the_30_entries_are_the_largest(built_library):
    def plan(n=1, width=1, tokens=1):
        return built_library.i4mm_cache_plan(n, 16, 16, 16, width, width, 16, 1, 16, 16, tokens, *(16,) * 6, None)
    assert plan(tokens=2 ** 30 + 1) == capi.ERR_SHAPE and plan(tokens=2 ** 31 - 4097) == capi.ERR_SHAPE
    assert plan(n=16384, width=2 ** 16 + 1) == capi.ERR_SHAPE and plan(n=2, width=2 ** 30) == capi.ERR_SHAPE and plan(n=16384, width=2 ** 31 - 1) == capi.ERR_SHAPE


def test_strides_of_a_single_page_head_or_token(built_library):
    """They lead nowhere, so that any value is fine, the odd ones that slices and views come with among them."""
    lib = built_library
    if torch.cuda.is_available():
        pytest.skip("a call that is not refused would be launched")

    def accepted(status):
        return status not in (capi.ERR_ALIGN, capi.ERR_SHAPE)

    def cache(pages=4, heads=2, **strides):
        s = dict(k_page=4096, k_head=2048, k_token=128, v_page=4096, v_head=2048, v_token=128)
        s.update(strides)
        return ctypes.byref(capi.Cache(16, 16, 16, pages, heads, 16, 128, *(s[n] for n in ("k_page", "k_head", "k_token", "v_page", "v_head", "v_token")), 0))

    def calls(c, heads, token=128 * 4, head=128, tokens=1):
        return (lib.i4mm_cache_write(c, 16, 16, 0, tokens, token, head, token, head, 16, None), lib.i4mm_cache_read(c, 16, 16, 0, tokens, 16, None),
                lib.i4mm_cache_attention(c, 16, 16, 0, tokens, heads, token, head, 16, 1, 1, 16, None, 1, 1, 1.0, 0, 16, 1 << 30, None))
    for odd in (1, 0, -3, 2 ** 40 + 1):
        assert all(map(accepted, calls(cache(heads=1, k_head=odd, v_head=odd), 1))), odd
        assert all(map(accepted, calls(cache(pages=1, k_page=odd, v_page=odd), 2))), odd
        assert all(map(accepted, calls(cache(), 2, token=odd))), odd
        assert all(map(accepted, calls(cache(heads=1), 1, head=odd))), odd
    for heads, strides in ((1, dict(k_page=4097)), (2, dict(v_head=1)), (1, dict(k_token=72)), (1, dict(v_page=-16)), (2, dict(k_head=2 ** 31))):
        assert not any(map(accepted, calls(cache(heads=heads, **strides), heads))), strides
    write, _, attend = calls(cache(), 2, head=4)
    assert write == attend == capi.ERR_ALIGN
    write, _, attend = calls(cache(heads=1), 1, token=4, tokens=2)
    assert write == attend == capi.ERR_ALIGN


def test_the_widest_block_table(built_library):
    """Tiles of up to 128 tokens are counted in 32 bits: their last one has to end below 2^31."""
    def attend(page, width):
        c = capi.Cache(16, 16, 16, 4, 1, page, 128, page * 128, 128, 128, page * 128, 128, 128, 0)
        return built_library.i4mm_cache_attention(ctypes.byref(c), 16, 16, 0, 1, 1, 128, 128, 16, width, width, 16, None, 1, 1, 1.0, 0, 16, 0, None)
    for page in (16, 32, 64, 128):
        assert attend(page, (2 ** 31 - 128) // page) == capi.ERR_WORKSPACE             # (accepted: the next check is the scratch's)
        assert attend(page, (2 ** 31 - 128) // page + 1) == capi.ERR_SHAPE
