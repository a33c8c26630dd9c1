"""GPU: queries and keys normed, rotated and written in one launch, against 64 bits and against the writer."""
import pytest
import torch

from int4matmul_kernels_b200 import cache, ops
from shared_reference import turned, turned_bound

pytestmark = pytest.mark.gpu
INT8, E4M3 = torch.int8, torch.float8_e4m3fn
FP16, BF16 = torch.float16, torch.bfloat16


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def empty_cache(pages, heads, page, dim, held, seed=0):
    """Arrays full of bytes, scales of all sizes."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    k, v = (torch.randint(-120, 120, (pages, heads, page, dim), dtype=INT8, device="cuda", generator=gen).view(held) for _ in range(2))
    return k, v, torch.exp2(torch.randint(-9, -3, (pages, heads, 2), device="cuda", generator=gen).float())


def slots_of(held, new, page, seed):
    """Slots of requests with `held` tokens and `new` more, in pages of no order; and the number of pages."""
    gen = torch.Generator().manual_seed(seed)
    counts = [-(-(c + n) // page) for c, n in zip(held, new)]
    ids, out = torch.randperm(sum(counts) + 2, generator=gen).tolist(), []
    for c, n, count in zip(held, new, counts):
        mine = [ids.pop() for _ in range(count)]
        out += [mine[p // page] * page + p % page for p in range(c, c + n)]
    return out, sum(counts) + 2


def same_bytes(a, b):
    return torch.equal(a.view(INT8), b.view(INT8))


def check(held, new, hq, hkv, dim, page, kind, dtype, pairs, interleaved, norm, seed, pad=0, size=1.0, farthest=100000):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    slots, pages = slots_of(held, new, page, seed)
    tokens = len(slots) + pad
    slots = ints(slots + [-1] * pad)
    wide = (torch.randn((tokens, hq + 2 * hkv, dim), device="cuda", generator=gen) * size).to(dtype)
    q, k, v = wide[:, :hq], wide[:, hq:hq + hkv], wide[:, hq + hkv:]
    positions = torch.randint(0, farthest, (tokens,), device="cuda", generator=gen, dtype=torch.int32)
    table = cache.angles(positions, (10000.0 ** (-torch.arange(pairs, device="cuda", dtype=torch.float64) / pairs)).float()) if pairs else None
    qw, kw = ((1 + 0.3 * torch.randn(dim, device="cuda", generator=gen)).to(dtype) if norm else None for _ in range(2))
    kc, vc, scales = empty_cache(pages, hkv, page, dim, kind, seed)
    other = [t.clone() for t in (kc.view(INT8), vc.view(INT8), scales)]
    other = [other[0].view(kind), other[1].view(kind), other[2]]
    got = cache.append(kc, vc, scales, q, k, v, slots, table, q_weight=qw, k_weight=kw, eps=1e-5, interleaved=interleaved)
    assert got.shape == q.shape and got.dtype == dtype and got.is_contiguous()
    out, parts = turned(q, qw, table, 1e-5, interleaved)
    off, limit = (got.double() - out).abs(), turned_bound(out, parts, dtype)
    assert (off <= limit).all(), (off / limit).max().item()
    # keys are treated as queries are, and then written: to the byte
    spare = [t.clone() for t in (other[0].view(INT8), other[1].view(INT8), other[2])]
    turned_k = cache.append(spare[0].view(kind), spare[1].view(kind), spare[2], k, k, v, slots, table, q_weight=kw, k_weight=kw, eps=1e-5, interleaved=interleaved)
    out, parts = turned(k, kw, table, 1e-5, interleaved)
    assert ((turned_k.double() - out).abs() <= turned_bound(out, parts, dtype)).all()
    cache.write(*other, turned_k, v, slots)
    assert same_bytes(kc, other[0]) and same_bytes(vc, other[1]) and torch.equal(scales, other[2])
    return got


@pytest.mark.parametrize("kind,dtype", [(INT8, FP16), (INT8, BF16), (E4M3, FP16), (E4M3, BF16)])
@pytest.mark.parametrize("dim,pairs,interleaved,norm", [(64, 32, False, True), (64, 16, True, False), (64, 8, False, True), (128, 64, False, True),
                                                        (128, 64, True, True), (128, 32, False, False), (128, 24, False, True), (128, 40, True, True),
                                                        (128, 0, False, True), (64, 24, False, False)])
def test_forms(dim, pairs, interleaved, norm, kind, dtype):
    check([0, 15, 16, 3, 100], [1, 2, 17, 40, 1], 5, 3, dim, 16, kind, dtype, pairs, interleaved, norm, dim + pairs)


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (40, 40), (32, 8), (71, 1), (4, 3)])
def test_heads_and_pages(hq, hkv, page):
    check([0, 5, 127, 200], [130, 1, 2, 300], hq, hkv, 128, page, INT8, FP16, 64, False, True, page + hq, pad=3)
    check([0, 5, 63], [33, 1, 90], hq, hkv, 64, page, E4M3, BF16, 32, True, True, page + hq)


@pytest.mark.parametrize("tokens", [1, 2, 3, 1023, 1024, 1025, 1040, 1041, 3001])
def test_token_counts(tokens):
    check([7], [tokens], 4, 2, 128, 32, INT8, BF16, 64, False, True, tokens)


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("dim,pairs,interleaved,norm,kind,dtype", [(128, 64, False, True, INT8, FP16), (128, 32, True, True, E4M3, BF16), (64, 32, False, True, E4M3, FP16),
                                                                   (64, 8, True, False, INT8, BF16), (128, 0, False, True, INT8, FP16), (64, 0, False, True, E4M3, BF16)])
def test_many_tokens(dim, pairs, interleaved, norm, kind, dtype, page):
    """Prompts that begin anywhere in a page, single tokens and drafts between them, padding behind."""
    held = [0, 5, 127, 200, 31, 16, 15, 3, 0, 64, 90, 1]
    new = [900, 1, 333, 1, 2, 1, 1, 5, 17, 700, 129, 40]
    check(held, new, 7, 3, dim, page, kind, dtype, pairs, interleaved, norm, page + dim, pad=21)


@pytest.mark.parametrize("tokens", [60, 1500])
@pytest.mark.parametrize("kind,dtype", [(INT8, FP16), (E4M3, BF16)])
def test_infinities_among_many_tokens(kind, dtype, tokens):
    """Held as a write of the same keys and values holds them, with few tokens and with many, in runs and alone."""
    gen = torch.Generator(device="cuda").manual_seed(tokens)
    slots, pages = slots_of([3, 0, 40, 9, 7], [tokens, 1, 1, 50, 1], 32, 2)
    n = len(slots)
    q, k, v = torch.randn((3, n, 4, 128), device="cuda", generator=gen).to(dtype).unbind(0)
    for x in (k, v):
        for i, token in enumerate((0, 5, 17, 40, tokens - 1, tokens, tokens + 1, tokens + 9, n - 1)):
            x[token, i % 4, (31 * i) % 128] = (float("inf"), float("-inf"), float("nan"))[i % 3]
    table = cache.angles(torch.arange(n, dtype=torch.int32, device="cuda"), torch.ones(64, device="cuda"))
    a, b, spare = (empty_cache(pages, 4, 32, 128, kind, 3) for _ in range(3))
    cache.append(*a, q, k, v, ints(slots), table)
    turned_k = cache.append(*spare, k, k, v, ints(slots), table)
    cache.write(*b, turned_k, v, ints(slots))
    assert same_bytes(a[0], b[0]) and same_bytes(a[1], b[1]) and torch.equal(a[2], b[2])


@pytest.mark.parametrize("size", [0.0, 1e-4, 1.0, 300.0])
def test_sizes(size):
    for norm in (True, False):
        check([2, 40], [5, 20], 3, 2, 128, 16, INT8, FP16, 64, False, norm, 5, size=size)
        check([2, 40], [5, 20], 3, 2, 128, 16, E4M3, BF16, 64, True, norm, 5, size=size)


def test_only_queries_or_keys_are_normed():
    gen = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn((3, 2, 64), device="cuda", generator=gen).half() for _ in range(3))
    w, table = torch.full((64,), 2.0, device="cuda").half(), cache.angles(ints([1, 2, 3]), torch.ones(32, device="cuda"))
    for qw, kw, angles in ((w, None, table), (None, w, table), (w, None, None), (None, None, table)):
        held = empty_cache(1, 2, 16, 64, INT8)
        got = cache.append(*held, q, k, v, ints([0, 1, 2]), angles, q_weight=qw, k_weight=kw)
        out, parts = turned(q, qw, angles, 1e-6, False)
        assert ((got.double() - out).abs() <= turned_bound(out, parts, FP16)).all()
        kk = cache.read(*held, ints([0, 1, 2]))[0]
        out, _ = turned(k, kw, angles, 1e-6, False)
        # half a step of int8 in the page's scale, which is at most 2 / 127 of the largest, after one rounding to fp16
        assert ((kk.double() - out).abs() <= out.abs().amax((0, 2), keepdim=True) * (1 / 127 + 2.0 ** -9)).all()


def test_rotation_by_nothing_is_a_write():
    """Angles of position 0: queries come back, the cache gets what a write puts there, infinities and NaN among it."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    for dtype in (FP16, BF16):
        q, k, v = torch.randn((3, 70, 4, 128), device="cuda", generator=gen).to(dtype).unbind(0)
        for x in (q, k, v):                              # (a rotation mixes the values of a pair: both are the same here)
            x[3, 1, 5] = x[3, 1, 69] = float("inf")
            x[9, 0, 7] = x[9, 0, 71] = float("nan")
            x[20:25] = 0
        k[3, 1], k[9, 0] = 1.0, 1.0                      # inf * 0 is NaN in a rotation
        slots = ints(list(range(32, 96)) + [-1] * 6)
        table = cache.angles(torch.zeros(70, dtype=torch.int32, device="cuda"), torch.ones(64, device="cuda"))
        for kind in (INT8, E4M3):
            a, b = empty_cache(6, 4, 32, 128, kind, 3), empty_cache(6, 4, 32, 128, kind, 3)
            got = cache.append(*a, q, k, v, slots, table)
            cache.write(*b, k, v, slots)
            assert same_bytes(a[0], b[0]) and same_bytes(a[1], b[1]) and torch.equal(a[2], b[2])
            there = torch.ones(70, 4, dtype=torch.bool, device="cuda")
            there[3, 1] = there[9, 0] = False
            assert torch.equal(got[there], q[there]) and got[9, 0].isnan().any() and not got[3, 1].isfinite().all()


def test_infinite_keys_are_held_as_the_writer_holds_them():
    """Without a rotation: a norm of an infinite head is NaN there and 0 elsewhere, and NaN is held as 0."""
    k = torch.ones((16, 2, 64), dtype=FP16, device="cuda")
    k[4, 0, 9] = float("inf")
    k[5, 1, 3] = float("nan")
    w = torch.ones(64, dtype=FP16, device="cuda")
    held = empty_cache(2, 2, 16, 64, INT8)
    got = cache.append(*held, k, k, k, ints(list(range(16))), None, q_weight=w, k_weight=w)
    other = empty_cache(2, 2, 16, 64, INT8)
    cache.write(*other, got, k, ints(list(range(16))))
    assert same_bytes(held[0], other[0]) and torch.equal(held[2], other[2])
    kk = cache.read(*held, ints([4, 5]))[0]
    assert (kk[0, 0] == 0).all() and (kk[1, 1] == 0).all() and (kk[0, 1] != 0).all()


def test_padding_is_not_written():
    held = empty_cache(3, 2, 16, 64, INT8)
    before = [t.clone() for t in held]
    q = torch.randn((5, 4, 64), device="cuda").half()
    got = cache.append(*held, q, q[:, :2], q[:, 2:], ints([-1, -1, 48, 1000, -1, 7, 8]), cache.angles(ints([-1] * 5), torch.ones(32, device="cuda")))
    assert torch.equal(got, q) and all(torch.equal(a, b) for a, b in zip(held, before))
    assert cache.append(*held, q[:0], q[:0, :2], q[:0, 2:], ints([]), q_weight=q[0, 0].contiguous()).shape == (0, 4, 64)


def test_streams_graphs_and_modes():
    q, k, v = torch.randn((3, 9, 4, 128), device="cuda").half().unbind(0)
    slots, positions, freqs = ints(list(range(9))), ints(list(range(9))), torch.ones(64, device="cuda")
    held = empty_cache(2, 4, 16, 128, INT8)
    want = cache.append(*held, q, k, v, slots, cache.angles(positions, freqs))
    side, other = torch.cuda.Stream(), empty_cache(2, 4, 16, 128, INT8)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.inference_mode():
        got = cache.append(*other, q, k, v, slots, cache.angles(positions, freqs))
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want) and same_bytes(held[0], other[0])
    graph, third = torch.cuda.CUDAGraph(), empty_cache(2, 4, 16, 128, INT8)
    with torch.cuda.graph(graph):
        got = cache.append(*third, q, k, v, slots, cache.angles(positions, freqs))
    q *= 2
    positions += 5
    graph.replay()
    again = cache.append(*empty_cache(2, 4, 16, 128, INT8), q, k, v, slots, cache.angles(positions, freqs))
    assert torch.equal(got, again) and not torch.equal(got, want)


def test_refusals():
    q, k, v = torch.randn((3, 4, 2, 64), device="cuda").half().unbind(0)
    held, slots, table, w = empty_cache(2, 2, 16, 64, INT8), ints([0, 1, 2, 3]), cache.angles(ints([0] * 4), torch.ones(32, device="cuda")), q[0, 0].contiguous()
    good = dict(q=q, k=k, v=v, slots=slots, angles=table, q_weight=w, k_weight=w)
    cache.append(*held, **good)
    for error, bad in ((ValueError, dict(angles=None, q_weight=None, k_weight=None)), (ValueError, dict(slots=slots[:3])), (ValueError, dict(angles=table[:3])),
                       (TypeError, dict(angles=table.half())), (TypeError, dict(angles=table.cpu())), (ValueError, dict(q=q[:3])), (ValueError, dict(v=v[:, :1])),
                       (ValueError, dict(k=k[:, :1], v=v[:, :1])), (ValueError, dict(q=q.bfloat16())), (TypeError, dict(k=k.float())), (ValueError, dict(q_weight=w[:32])),
                       (ValueError, dict(k_weight=w.float())), (ValueError, dict(q_weight=w.cpu())), (ValueError, dict(angles=table[..., :1])),
                       (ValueError, dict(angles=table.transpose(0, 1)[:4])), (TypeError, dict(slots=slots.long())), (ValueError, dict(q=q[..., ::2])),
                       (ops.Int4MatmulError, dict(angles=torch.zeros((4, 4, 2), device="cuda"))), (ops.Int4MatmulError, dict(angles=torch.zeros((4, 40, 2), device="cuda"))),
                       (ops.Int4MatmulError, dict(q=torch.empty(4 * 128 + 8, device="cuda", dtype=FP16)[4:516].view(4, 2, 64)))):
        with pytest.raises(error):
            cache.append(*held, **{**good, **bad})
