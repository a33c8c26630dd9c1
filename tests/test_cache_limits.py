"""CPU: sizes whose loops would pass 32 bits are refused before anything touches a device, and strides that mean nothing are not."""
import ctypes

import torch

from int4matmul_kernels_b200 import capi


def test_tables_of_a_step_of_2_to_the_30_entries_are_the_largest(built_library):
    def plan(n=1, width=1, tokens=1):
        return built_library.i4mm_cache_plan(n, 16, 16, 16, width, width, 16, 1, 16, 16, tokens, *(16,) * 6, None)
    assert plan(tokens=2 ** 30 + 1) == capi.ERR_SHAPE and plan(tokens=2 ** 31 - 4097) == capi.ERR_SHAPE
    assert plan(n=16384, width=2 ** 16 + 1) == capi.ERR_SHAPE and plan(n=2, width=2 ** 30) == capi.ERR_SHAPE and plan(n=16384, width=2 ** 31 - 1) == capi.ERR_SHAPE
