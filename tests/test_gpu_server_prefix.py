"""GPU: the layer stack with positions and shared prefixes: every operator's result on the inputs it received, and the step as a whole."""
import math

import pytest
import torch

from cache_reference import attention_bound, values
from int4matmul_kernels_b200 import cache, serving, sharding
from shared_reference import attention as reference, share as share_reference, turned, turned_bound

pytestmark = pytest.mark.gpu
FREQS = 10000.0 ** (-torch.arange(0, 32, dtype=torch.float32) / 32)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def server(heads=4, dtype=torch.int8, window=0, pages=60, interleaved=False, norm=True):
    cfg = sharding.StackConfig(hidden=256, mlp=512, layers=3, bits=4, group_size=64)
    pairs = 256 // heads // 2
    return serving.CachedStack(sharding.DecoderStack(cfg, 0, 1, "cuda"), heads, pages, 16, 5, 160, dtype, window, FREQS[:pairs].cuda(), norm, interleaved)


# place 0 becomes the prefix of 1, 2 and 4; 3 has none, and is one itself for 2 later
STEPS = [([37, 0, 0, 20, 0], None), ([0, 11, 3, 1, 70], [-1, 0, 0, -1, 0]), ([0, 1, 1, 1, 1], [-1, 0, 0, -1, 0]), ([0, -1, 1, 1, 1], [-1, 0, 0, -1, 0]),
         ([0, 5, -1, 0, 2], [-1, 0, -1, -1, 0]), ([0, 1, 9, 0, 1], [-1, 0, 3, -1, 0]), ([2, 1, 1, 1, 1], [-1, 0, 3, -1, 0])]


@pytest.mark.parametrize("heads,dtype,window,interleaved,norm", [(4, torch.int8, 0, False, True), (2, torch.float8_e4m3fn, 0, True, False), (4, torch.int8, 24, True, True)])
def test_steps_of_a_server(heads, dtype, window, interleaved, norm, monkeypatch):
    s = server(heads, dtype, window, interleaved=interleaved, norm=norm)
    seen, turns = [], []
    attend, append = cache.attention, cache.append

    def recorded(q, k, v, scales, table, seq, cu, max_len, *, scale=None, window=0, **more):
        out = attend(q, k, v, scales, table, seq, cu, max_len, scale=scale, window=window, **more)
        seen.append((q.clone(), values(k, scales[..., 0]), values(v, scales[..., 1]), table.clone(), seq.clone(), cu.clone(), more, window, out.clone()))
        return out

    def recorded_append(kc, vc, scales, q, k, v, slots, angles, **more):
        out = append(kc, vc, scales, q, k, v, slots, angles, **more)
        turns.append((q.clone(), angles.clone(), more, out.clone()))
        return out
    monkeypatch.setattr(cache, "attention", recorded)
    monkeypatch.setattr(cache, "append", recorded_append)
    gen = torch.Generator(device="cuda").manual_seed(3)
    for new, of in STEPS:
        tokens = sum(max(n, 0) for n in new)
        h = torch.randn((tokens, 256), device="cuda", generator=gen).half()
        seen.clear()
        turns.clear()
        out = s.step(h, ints(new), max(new), None if of is None else ints(of))
        assert out.shape == h.shape and torch.isfinite(out).all() and len(seen) == len(turns) == 3 and s.plan.missing.item() == 0
        cu = [0]
        for n in new:
            cu.append(cu[-1] + max(n, 0))
        want = share_reference(of or [-1] * 5, s.table.seq_lens.tolist(), cu, tokens)
        a = torch.tensor(want["positions"], dtype=torch.float64, device="cuda")[:, None] * s.freqs.double()
        for q, angles, more, got in turns:
            assert ((angles.double() - torch.stack([a.cos(), a.sin()], -1)).abs() < 1e-6).all() and more["interleaved"] == interleaved
            o, size = turned(q, more["q_weight"], angles, 1e-6, interleaved)
            assert (more["q_weight"] is not None) == norm and ((got.double() - o).abs() <= turned_bound(o, size, q.dtype)).all()
        for q, k, v, t, sl, c, more, w, got in seen:
            assert w == window and c.tolist() == cu and ("shared" in more) == (of is not None)
            o, size, reach, tail = reference(q, k, v, t, sl, c, want["prefix_of"], 1 / math.sqrt(256 // heads), w)
            assert ((got.double() - o).abs() <= attention_bound(o, size, reach, tail, q.dtype)).all()


@pytest.mark.parametrize("window", [0, 30])
def test_sharing_changes_nothing_but_the_cache_s_rounding(window):
    """37 tokens held once for three requests, and held by each of them: rows see the same tokens at the same positions; only the pages' scales differ, by
    less than a step of a 7-bit value, 1 / 64 of a page's largest."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    prefix = torch.randn((37, 256), device="cuda", generator=gen).half()
    own = [torch.randn((n, 256), device="cuda", generator=gen).half() for n in (11, 1, 40)]
    s, whole = server(window=window), server(window=window)
    s.step(prefix, ints([37, 0, 0, 0, 0]), 37)
    of = ints([-1, 0, 0, 0, -1])
    got = s.step(torch.cat(own), ints([0, 11, 1, 40, 0]), 40, of)
    want = whole.step(torch.cat([torch.cat([prefix, x]) for x in own]), ints([0, 48, 38, 77, 0]), 77)
    want = torch.cat([want[37:48], want[85:86], want[123:163]])
    assert (got.double() - want.double()).norm() / want.double().norm() < 3 * 1 / 64
    x = torch.randn((3, 256), device="cuda", generator=gen).half()
    got, want = s.step(x, ints([0, 1, 1, 1, 0]), 1, of), whole.step(x, ints([0, 1, 1, 1, 0]), 1)
    assert (got.double() - want.double()).norm() / want.double().norm() < 3 * 1 / 64
    # and they do see it
    other = server(window=window)
    other.step(prefix, ints([37, 0, 0, 0, 0]), 37)
    assert (other.step(x, ints([0, 1, 1, 1, 0]), 1).double() - got.double()).norm() / got.double().norm() > 0.1


def test_a_step_in_a_graph():
    """A captured step of requests under a prefix serves every later one."""
    gen = torch.Generator(device="cuda").manual_seed(6)
    plain, captured = server(), server()
    prefix, of = torch.randn((37, 256), device="cuda", generator=gen).half(), ints([-1, 0, -1, 0, 0])
    prompts, new = torch.randn((52, 256), device="cuda", generator=gen).half(), ints([0, 20, 30, 1, 1])
    for s in (plain, captured):
        s.step(prefix, ints([37, 0, 0, 0, 0]), 37)
        s.step(prompts, new, 30, of)
    h, ones = torch.zeros((4, 256), dtype=torch.float16, device="cuda"), ints([0, 1, 1, 1, 1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = captured.step(h, ones, 1, of)
    for _ in range(20):
        x = torch.randn((4, 256), device="cuda", generator=gen).half()
        h.copy_(x)
        graph.replay()
        assert torch.equal(plain.step(x, ones, 1, of), out)
    assert plain.table.seq_lens.tolist() == captured.table.seq_lens.tolist()


def test_a_step_short_of_pages_is_not_made():
    s = server(pages=5)
    s.step(torch.randn((37, 256), device="cuda").half(), ints([37, 0, 0, 0, 0]), 37)
    before = [t.clone() for c in s.caches for t in (c.k, c.v, c.scales)]
    s.step(torch.randn((60, 256), device="cuda").half(), ints([0, 30, 30, 0, 0]), 30, ints([-1, 0, 0, -1, -1]))
    assert s.plan.missing.item() > 0 and s.table.seq_lens.tolist() == [37, 0, 0, 0, 0]
    assert all(torch.equal(a, b) for a, b in zip(before, [t for c in s.caches for t in (c.k, c.v, c.scales)]))
    out = s.step(torch.randn((3, 256), device="cuda").half(), ints([0, 1, 2, 0, 0]), 2, ints([-1, 0, 0, -1, -1]))
    assert s.plan.missing.item() == 0 and torch.isfinite(out).all()


def test_refusals():
    cfg = sharding.StackConfig(hidden=256, mlp=512, layers=1, bits=4, group_size=64)
    stack = sharding.DecoderStack(cfg, 0, 1, "cuda")
    for freqs in (FREQS.cuda().double(), FREQS, FREQS[:12].cuda(), torch.ones(40, device="cuda"), FREQS[None].cuda(), FREQS[:0].cuda()):
        with pytest.raises(ValueError):
            serving.CachedStack(stack, 4, 4, 16, 1, 64, freqs=freqs)
    s = server()
    h = torch.zeros((1, 256), dtype=torch.float16, device="cuda")
    for of in (ints([-1] * 4), ints([-1] * 5).long(), ints([-1] * 5).cpu(), ints([-1] * 10)[::2]):
        with pytest.raises(ValueError):
            s.step(h, ints([1, 0, 0, 0, 0]), 1, of)
    assert s.table.seq_lens.tolist() == [0] * 5
