"""GPU: scratch that is first used in inference mode is cleared after a time-out like any other."""
import pytest
import torch

from int4matmul_kernels_b200 import cache, capi, ops

pytestmark = pytest.mark.gpu
STATUS = 256 * 1024 - 64


def attention():
    c = cache.PagedCache(2, 1, 16, 64)
    x = torch.zeros((1, 1, 64), dtype=torch.float16, device="cuda")
    one = torch.ones(1, dtype=torch.int32, device="cuda")
    return lambda: cache.attention(x, c.k, c.v, c.scales, (one - 1)[None], one)


def multiply():
    matrix = torch.zeros((16, 64), dtype=torch.int32, device="cuda")
    ones, x = (torch.ones(s, dtype=torch.float16, device="cuda") for s in ((1, 64), (1, 1, 128)))
    out = torch.zeros((1, 1, 64), dtype=torch.float16, device="cuda")
    return lambda: ops.quant_matmul(4, out, matrix, x, ones, ones, 128, None)


@pytest.mark.parametrize("make,scratch", [(attention, "_cache_workspaces"), (multiply, "_workspaces")])
def test_a_time_out_of_scratch_made_in_inference_mode(make, scratch, monkeypatch):
    monkeypatch.setattr(ops, scratch, {})
    with torch.inference_mode():
        make()()
        (ws,) = getattr(ops, scratch).values()
        ws[STATUS], ws[0] = 61, 7                               # as a kernel that gave up leaves it
    with pytest.raises(ops.Int4MatmulError) as e:
        ops.check_device_status()
    assert e.value.status == capi.ERR_TIMEOUT and not ws.any()
    ops.check_device_status()
