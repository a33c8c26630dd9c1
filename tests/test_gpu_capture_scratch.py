"""GPU: scratch whose first use is in a graph capture belongs to no graph: graphs of one stream may be replayed in any order, none of them clears
it, and what a kernel has recorded in it stays until it is read."""
import pytest
import torch

import int4matmul_kernels_b200 as package
from int4matmul_kernels_b200 import cache, capi, ops

pytestmark = pytest.mark.gpu
STATUS = 256 * 1024 - 64


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def graph_of(stream, call):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = call()
    return graph, out


def memory_of(graph):
    """bytes of the graph's private pool"""
    return sum(s["total_size"] for s in torch.cuda.memory_snapshot() if tuple(s["segment_pool_id"]) == tuple(graph.pool()))


def check(calls, scratch_bytes):
    """calls: each returns its result; none has run on `stream` before"""
    want = [c().clone() for c in calls]
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    made = [graph_of(stream, c) for c in calls]
    assert all(memory_of(g) < scratch_bytes for g, _ in made)
    for g, out in made:
        out.zero_()
    for g, out in reversed(made):
        g.replay()
    torch.cuda.synchronize()
    for (_, out), w in zip(made, want):
        assert torch.equal(out, w)
    return stream, made


def status_stays(scratch, stream, made):
    ws = scratch[(torch.cuda.current_device(), stream.cuda_stream)]
    ws[STATUS] = 61                                          # as a kernel that gave up leaves it
    for g, _ in made:
        g.replay()
    with pytest.raises(ops.Int4MatmulError) as e:
        ops.check_device_status()
    assert e.value.status == capi.ERR_TIMEOUT
    ops.check_device_status()


@pytest.mark.parametrize("compiled", [True, False])
def test_attention(compiled, monkeypatch):
    monkeypatch.setattr(ops, "_cache_workspaces", {})
    if not compiled:
        monkeypatch.setattr(ops, "_native", False)
    gen = torch.Generator(device="cuda").manual_seed(1)
    c, table = cache.PagedCache(300, 2, 16, 128), cache.PageTable(2, 300, 16, 4000)
    p = table.step(ints([3000, 900]), 3900)
    x = torch.randn((3900, 8, 128), device="cuda", generator=gen).half()
    c.write(x[:, :2], x[:, 2:4], p.slots)
    few = lambda: c.attention(x[:2], table)                                        # noqa: E731
    many = lambda: c.attention(x, table, p.cu_lens, 3000)                          # noqa: E731
    stream, made = check([few, many, few], capi.load().i4mm_cache_attention_workspace_bytes())
    status_stays(ops._cache_workspaces, stream, made)


def problem(rows):
    gen = torch.Generator(device="cuda").manual_seed(rows)
    matrix = torch.randint(-2 ** 31, 2 ** 31 - 1, (128, 512), dtype=torch.int32, device="cuda", generator=gen)
    scales = (torch.rand((8, 512), device="cuda", generator=gen) * 0.01).half()
    zeros = torch.randint(0, 16, (8, 512), device="cuda", generator=gen).half()
    x = torch.randn((1, rows, 1024), device="cuda", generator=gen).half()
    out = torch.empty((1, rows, 512), dtype=torch.float16, device="cuda")
    return out, matrix, x, scales, zeros


@pytest.mark.parametrize("route", ["ops", "ops without the compiled module", "module"])
def test_multiplies(route, monkeypatch):
    monkeypatch.setattr(ops, "_workspaces", {})
    if "without" in route:
        monkeypatch.setattr(ops, "_native", False)
    entry = package.load_extension() if route == "module" else ops

    def multiply(rows):
        out, matrix, x, scales, zeros = problem(rows)

        def call():
            entry.quant_matmul(4, out, matrix, x, scales, zeros, 128, None)
            return out
        return call
    stream, made = check([multiply(r) for r in (48, 300, 12)], capi.load().i4mm_workspace_bytes())
    if route != "module":
        status_stays(ops._workspaces, stream, made)
