"""GPU: infinities in a page that holds nothing else but zeros, and values that follow them."""
import math

import pytest
import torch

from int4matmul_kernels_b200 import cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("held", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64)])
def test_a_scale_that_grows_from_nothing(dim, page, dtype, held):
    """The scale of such a page is 0, what it holds stands for 0, and stays so: round(q * old / s) with old = 0."""
    c = cache.PagedCache(2, 2, page, dim, held)
    x = torch.zeros((3, 4, dim), dtype=dtype, device="cuda")
    x[0, :, ::3], x[1, :, 1::5], x[2, 0] = math.inf, -math.inf, math.nan
    slots = torch.arange(4, dtype=torch.int32, device="cuda") + page
    c.write(x[:, :2], x[:, 2:], slots[:3])
    first = c.read(slots[:3], dtype)
    assert (c.scales == 0).all() and all((f == 0).all() for f in first)
    y = torch.randn((1, 4, dim), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(dtype)
    c.write(y[:, :2], y[:, 2:], slots[3:])
    assert (c.scales[1] > 0).all()
    for now, new in zip(c.read(slots, dtype), (y[:, :2], y[:, 2:])):
        assert (now[:3] == 0).all()
        assert ((now[3:] - new).abs().float() <= (1 / 64 if held == torch.int8 else 1 / 16) * new.abs().max().float()).all()
