"""GPU: the cache's calls where only the C ABI library is built (no compiled module), and its device status."""
import math

import pytest
import torch

from int4matmul_kernels_b200 import cache, capi, ops

pytestmark = pytest.mark.gpu


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def step(dtype, held):
    gen = torch.Generator(device="cuda").manual_seed(1)
    table = cache.PageTable(3, 30, 16, 128)
    c = cache.PagedCache(30, 2, 16, 64, held)
    results = []
    for new in ([20, 1, 0], [1, 1, 50], [1, -1, 1]):
        tokens = sum(max(n, 0) for n in new)
        p = table.step(ints(new), tokens + 2)
        x = torch.randn((tokens, 8, 64), device="cuda", generator=gen).to(dtype)
        c.write(x[:, 4:6], x[:, 6:], p.slots)
        results += [*p, *c.read(p.slots, dtype), c.attention(x[:, :4], table, p.cu_lens, max(new)), c.scales.clone(), c.k.view(torch.int8).clone()]
    return results


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("held", [torch.int8, torch.float8_e4m3fn])
def test_both_ways_give_the_same(dtype, held, monkeypatch):
    compiled = step(dtype, held)
    monkeypatch.setattr(ops, "_native", False)
    for a, b in zip(compiled, step(dtype, held)):
        assert torch.equal(a, b)


def test_refusals_without_the_compiled_module(monkeypatch):
    monkeypatch.setattr(ops, "_native", False)
    c = cache.PagedCache(4, 2, 16, 64)
    x = torch.zeros((3, 2, 64), dtype=torch.float16, device="cuda")
    with pytest.raises(TypeError):
        c.write(x.float(), x, ints([0, 1, 2]))
    with pytest.raises(ValueError):
        c.write(x, x, ints([0, 1]))
    with pytest.raises(ValueError):
        cache.attention(x, c.k, c.v, c.scales, ints([[0]]), ints([1, 2]))
    with pytest.raises(ops.Int4MatmulError) as e:
        cache.plan(ints([1]), ints([1]), ints([[0]]), ints([1]), ints([1]), 17, 1)
    assert e.value.status == capi.ERR_UNSUPPORTED
    assert math.isfinite(float(c.scales.sum()))


def test_device_status_covers_the_attention_scratch():
    c, table = cache.PagedCache(4, 2, 16, 64), cache.PageTable(1, 4, 16, 64)
    p = table.step(ints([30]), 30)
    x = torch.randn((30, 2, 64), device="cuda").half()
    c.write(x, x, p.slots)
    c.attention(x, table, p.cu_lens, 30)
    ops.check_device_status()
    stream = torch.cuda.current_stream()
    ws = ops._cache_workspaces[(torch.cuda.current_device(), stream.cuda_stream)]
    status = 256 * 1024 - 64
    ws[status] = 61                                              # as a kernel that gave up leaves it
    with pytest.raises(ops.Int4MatmulError) as e:
        ops.check_device_status()
    assert e.value.status == capi.ERR_TIMEOUT
    ops.check_device_status()
    c.attention(x, table, p.cu_lens, 30)
    ops.check_device_status()
