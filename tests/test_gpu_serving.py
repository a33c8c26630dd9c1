"""GPU: the layer stack over the paged cache, requests coming and going: every operator's result on the inputs it received."""
import math

import pytest
import torch

from cache_reference import attention as reference, attention_bound, plan as plan_reference, values
from int4matmul_kernels_b200 import cache, serving, sharding

pytestmark = pytest.mark.gpu


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def server(heads=4, dtype=torch.int8, window=0, pages=40):
    cfg = sharding.StackConfig(hidden=256, mlp=512, layers=3, bits=4, group_size=64)
    return serving.CachedStack(sharding.DecoderStack(cfg, 0, 1, "cuda"), heads, pages, 16, 5, 160, dtype, window)


STEPS = [[20, 3, 0, 1, 0], [1, 1, 0, 1, 40], [1, -1, 33, 1, 1], [1, 0, 1, 1, 1], [-1, 2, 1, 16, 1], [5, 1, 1, -1, 70]]


@pytest.mark.parametrize("heads,dtype,window", [(4, torch.int8, 0), (2, torch.float8_e4m3fn, 0), (4, torch.int8, 24)])
def test_steps_of_a_server(heads, dtype, window, monkeypatch):
    s = server(heads, dtype, window)
    seen = []
    plain = cache.attention

    def recorded(q, k, v, scales, table, seq, cu, max_len, *, scale=None, window=0):
        out = plain(q, k, v, scales, table, seq, cu, max_len, scale=scale, window=window)
        seen.append((q.clone(), values(k, scales[..., 0]), values(v, scales[..., 1]), table.clone(), seq.clone(), cu.clone(), window, out.clone()))
        return out
    monkeypatch.setattr(cache, "attention", recorded)
    gen = torch.Generator(device="cuda").manual_seed(3)
    seq, stack, table = [0] * 5, list(range(39, -1, -1)), [[-1] * 10 for _ in range(5)]
    for new in STEPS:
        tokens = sum(max(n, 0) for n in new)
        h = torch.randn((tokens, 256), device="cuda", generator=gen).half()
        seen.clear()
        out = s.step(h, ints(new), max(new))
        want = plan_reference(seq, new, table, stack, 16, 10, tokens)
        seq, table, stack = want["lens"], want["table"], want["pushed"][:want["free"]]
        assert s.table.seq_lens.tolist() == seq and s.table.block_table.tolist() == table and s.table.free_count.item() == len(stack)
        assert out.shape == h.shape and torch.isfinite(out).all() and len(seen) == 3
        for q, k, v, t, sl, cu, w, got in seen:
            assert w == window and cu.tolist() == want["cu"]
            o, size, reach, tail = reference(q, k, v, t, sl, cu, 1 / math.sqrt(256 // heads), w)
            assert ((got.double() - o).abs() <= attention_bound(o, size, reach, tail, q.dtype)).all()


def test_a_prompt_in_pieces_is_the_prompt_but_for_the_cache_s_rounding():
    """The same 60 tokens at once, and as 25 + 1 + 34: rows see the same tokens; only scales that grew in between differ, by less than a step
    of a 7-bit value, 1 / 64 of a page's largest."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    h = torch.randn((60, 256), device="cuda", generator=gen).half()
    whole = server().step(h, ints([60, 0, 0, 0, 0]), 60)
    s = server()
    parts = torch.cat([s.step(h[a:b], ints([b - a, 0, 0, 0, 0]), b - a) for a, b in ((0, 25), (25, 26), (26, 60))])
    off = (whole.double() - parts.double()).norm() / whole.double().norm()
    assert off < 3 * 1 / 64
    again = server().step(h, ints([60, 0, 0, 0, 0]), 60)
    assert torch.equal(again, whole)


def test_a_step_in_a_graph():
    """Tables, lengths and pages are on the GPU: a captured decoding step serves every later one."""
    gen = torch.Generator(device="cuda").manual_seed(6)
    plain, captured = server(), server()
    prompts, new = torch.randn((52, 256), device="cuda", generator=gen).half(), ints([20, 30, 1, 0, 1])
    for s in (plain, captured):
        s.step(prompts, new, 30)
    h, ones = torch.zeros((4, 256), dtype=torch.float16, device="cuda"), ints([1, 1, 1, 0, 1])
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):                               # (the stream's scratch exists before the capture)
        warm = server()
        warm.step(prompts, new, 30)
        warm.step(h, ones, 1)
    side.synchronize()
    t = captured.table
    seq, count = t.seq_lens, t.free_count
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = captured.step(h, ones, 1)
        seq.copy_(t.seq_lens)
        count.copy_(t.free_count)
    for _ in range(20):
        x = torch.randn((4, 256), device="cuda", generator=gen).half()
        h.copy_(x)
        graph.replay()
        assert torch.equal(plain.step(x, ones, 1), out)
    assert plain.table.seq_lens.tolist() == seq.tolist()


def test_refusals():
    cfg = sharding.StackConfig(hidden=256, mlp=512, layers=1, bits=4, group_size=64)
    stack = sharding.DecoderStack(cfg, 0, 1, "cuda")
    with pytest.raises(ValueError):
        serving.CachedStack(stack, 3, 4, 16, 1, 64)
    with pytest.raises(TypeError):
        serving.CachedStack(stack, 4, 4, 16, 1, 64, torch.float16)
    stack.world = 2
    with pytest.raises(ValueError):
        serving.CachedStack(stack, 4, 4, 16, 1, 64)
