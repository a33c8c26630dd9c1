"""GPU: the cache's writer and reader against 64 bits: the bytes and scales are equal, not near."""
import math

import pytest
import torch

from cache_reference import MOST, values, write_one
from int4matmul_kernels_b200 import cache, capi, ops

pytestmark = pytest.mark.gpu
INT8, E4M3 = torch.int8, torch.float8_e4m3fn


def empty(pages, heads, page, dim, dtype, order="heads"):
    """k, v, scales; order "tokens": (pages, page, heads, dim) in memory, "together": keys and values of a page side by side."""
    if order == "heads":
        k, v = (torch.zeros((pages, heads, page, dim), dtype=torch.int8, device="cuda") for _ in range(2))
    elif order == "tokens":
        k, v = (torch.zeros((pages, page, heads, dim), dtype=torch.int8, device="cuda").transpose(1, 2) for _ in range(2))
    else:
        k, v = torch.zeros((pages, heads, page, 2, dim), dtype=torch.int8, device="cuda").unbind(3)
    return k.view(dtype), v.view(dtype), torch.zeros((pages, heads, 2), device="cuda")


def held(c, s):
    """The cache's numbers in 64 bits, for the reference to work on."""
    return c.view(torch.int8).clone(memory_format=torch.contiguous_format).view(c.dtype).double().cpu(), s.double().cpu()


def step(k_cache, v_cache, scales, k, v, slots):
    """One write on both sides; asserts that the cache holds the same numbers."""
    page = k_cache.shape[2]
    want = [held(c, scales[..., i]) for i, c in enumerate((k_cache, v_cache))]
    for (h, s), x in zip(want, (k, v)):
        write_one(h, s, x.double().cpu(), slots.tolist(), page, k_cache.dtype)
    cache.write(k_cache, v_cache, scales, k, v, slots)
    for i, (c, (h, s)) in enumerate(zip((k_cache, v_cache), want)):
        got, gs = held(c, scales[..., i])
        assert torch.equal(gs, s)
        assert torch.equal(got, h), (i, (got != h).nonzero()[:4])


def rows(gen, tokens, heads, dim, dtype, spread=1.0):
    x = torch.randn((tokens, heads, dim), device="cuda", generator=gen) * torch.exp(spread * torch.randn((tokens, heads, 1), device="cuda", generator=gen))
    return x.to(dtype)


def slots_of(page, pages, runs, seed):
    """runs: (first place, tokens): laid over pages in a random order, as a plan lays out requests"""
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    out = []
    for first, n in runs:
        ids = [order.pop() for _ in range(-(-(first + n) // page))]
        out += [ids[p // page] * page + p % page for p in range(first, first + n)]
    return torch.tensor(out, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("order", ["heads", "tokens", "together"])
@pytest.mark.parametrize("held_as", [INT8, E4M3])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("page,dim,heads", [(16, 128, 5), (64, 64, 3), (128, 128, 1), (32, 64, 8)])
def test_steps_of_a_batch(page, dim, heads, dtype, held_as, order):
    """A prompt for some requests, then single tokens for all, then a few: partly filled pages, growing scales, odd lengths."""
    gen = torch.Generator(device="cuda").manual_seed(page + dim + heads)
    lens = [0, 1, page - 1, page, 2 * page + 3, 5, 3 * page]
    pages = 60
    k, v, scales = empty(pages, heads, page, dim, held_as, order)
    order_of = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).tolist()
    tables = [order_of[8 * b:8 * b + 8] for b in range(len(lens))]
    at = [0] * len(lens)
    for news in (lens, [1] * 7, [1] * 7, [3, 0, page, 1, 2, 1, page + 1], [1] * 7, [1] * 7):
        slots = []
        for b, n in enumerate(news):
            slots += [tables[b][p // page] * page + p % page for p in range(at[b], at[b] + n)]
            at[b] += n
        x = rows(gen, len(slots), 2 * heads, dim, dtype)
        step(k, v, scales, x[:, :heads], x[:, heads:], torch.tensor(slots, dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("tokens", [1, 2, 15, 16, 17, 33, 1000, 1024, 1025, 2500])
@pytest.mark.parametrize("held_as", [INT8, E4M3])
def test_token_counts(tokens, held_as):
    gen = torch.Generator(device="cuda").manual_seed(tokens)
    k, v, scales = empty(200, 3, 16, 64, held_as)
    first = tokens % 13
    x = rows(gen, tokens, 6, 64, torch.float16)
    slots = slots_of(16, 200, [(first, tokens)], tokens)
    step(k, v, scales, x[:, :3], x[:, 3:], slots)


@pytest.mark.parametrize("held_as", [INT8, E4M3])
def test_many_requests_of_a_few_tokens(held_as):
    gen = torch.Generator(device="cuda").manual_seed(4)
    k, v, scales = empty(1300, 2, 32, 128, held_as)
    runs = [((7 * i) % 32, 1 + (i * i) % 3) for i in range(600)]
    slots = slots_of(32, 1300, runs, 2)
    for n in (slots.shape[0], 700):
        x = rows(gen, n, 4, 128, torch.bfloat16)
        step(k, v, scales, x[:, :2], x[:, 2:], slots[:n].contiguous())


@pytest.mark.parametrize("held_as", [INT8, E4M3])
def test_padding_and_slots_outside(held_as):
    gen = torch.Generator(device="cuda").manual_seed(9)
    k, v, scales = empty(6, 2, 16, 64, held_as)
    slots = torch.tensor([-1, 16, 17, -1, 18, -5, 96, 97, 2 ** 31 - 1, 40, 41, -1], dtype=torch.int32, device="cuda")
    x = rows(gen, 12, 4, 64, torch.float16)
    # 18 follows a padded token: a run of its own in a page that the call has begun; kept apart here by writing it afterwards
    slots[4] = -1
    step(k, v, scales, x[:, :2], x[:, 2:], slots)
    step(k, v, scales, x[:1, :2], x[:1, 2:], torch.tensor([18], dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("held_as", [INT8, E4M3])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_zeros_infinities_nan_and_extremes(held_as, dtype):
    top = torch.finfo(dtype).max
    tiny = torch.finfo(dtype).tiny
    special = [0.0, -0.0, math.inf, -math.inf, math.nan, top, -top, tiny, -tiny, tiny / 4, 1.0, -1.0, 127.0, 127.5, 448.0, 449.0, 0.5, 2.0 ** -9]
    k, v, scales = empty(8, 1, 16, 64, held_as)
    for i, group in enumerate([special, [0.0], [math.inf], [math.nan, 1.0], [tiny / 4], [127.0], [448.0, -448.0, 1.0], [-math.inf, tiny]]):
        x = torch.zeros((3, 2, 64), dtype=dtype, device="cuda")
        x[:, 0] = torch.tensor([group[j % len(group)] for j in range(64)], device="cuda").to(dtype)
        x[1, 1] = x[0, 0].flip(0)
        slots = torch.arange(3, dtype=torch.int32, device="cuda") + 16 * i
        step(k, v, scales, x[:, :1], x[:, 1:], slots)
        step(k, v, scales, x[:, 1:] * 2, x[:, :1], slots + 3)


@pytest.mark.parametrize("held_as", [INT8, E4M3])
def test_error_of_a_token_after_its_page_grew_many_times(held_as):
    """Values that double with every token: each raises the scale; what is held is off by less than one step of the final scale."""
    k, v, scales = empty(1, 2, 64, 64, held_as)
    gen = torch.Generator(device="cuda").manual_seed(5)
    all_x = []
    for t in range(20):
        x = (torch.randn((1, 4, 64), device="cuda", generator=gen) * 2.0 ** (t - 10)).half()
        all_x.append(x)
        step(k, v, scales, x[:, :2], x[:, 2:], torch.tensor([t], dtype=torch.int32, device="cuda"))
    x = torch.cat(all_x).double()
    for i, c in enumerate((k, v)):
        got = values(c, scales[..., i])[0, :, :20].transpose(0, 1)
        off = (got - x[:, 2 * i:2 * i + 2]).abs()
        one = scales[0, :, i].double()[None, :, None]
        # e4m3: a step is 2^-3 of a value's power of two, one quantum (2^-9) at the least
        limit = one if held_as == INT8 else one * torch.maximum(torch.exp2(torch.floor(torch.log2((x[:, 2 * i:2 * i + 2].abs() / one).clamp(min=2.0 ** -6))) - 3) * 1.5,
                                                               torch.tensor(2.0 ** -9, device="cuda"))
        assert (off < limit).all()


def test_reused_page_begins_anew():
    gen = torch.Generator(device="cuda").manual_seed(6)
    k, v, scales = empty(2, 1, 16, 64, INT8)
    big, small = rows(gen, 16, 2, 64, torch.float16) * 100, rows(gen, 2, 2, 64, torch.float16) * 0.01
    slots = torch.arange(16, dtype=torch.int32, device="cuda")
    step(k, v, scales, big[:, :1], big[:, 1:], slots)
    step(k, v, scales, small[:, :1], small[:, 1:], slots[:2])
    assert float(scales[0].max()) < 0.01


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("held_as", [INT8, E4M3])
@pytest.mark.parametrize("order", ["heads", "tokens"])
def test_read_gives_what_the_bytes_stand_for(dtype, held_as, order):
    gen = torch.Generator(device="cuda").manual_seed(8)
    k, v, scales = empty(20, 3, 32, 128, held_as, order)
    x = rows(gen, 300, 6, 128, dtype, 0.3)
    slots = slots_of(32, 20, [(0, 300)], 3)
    cache.write(k, v, scales, x[:, :3], x[:, 3:], slots)
    pick = torch.cat([slots[::7], torch.tensor([-1, 640, 2 ** 31 - 1], dtype=torch.int32, device="cuda"), slots[:1]])
    got = cache.read(k, v, scales, pick, dtype)
    for i, c in enumerate((k, v)):
        all_ = values(c, scales[..., i]).transpose(1, 2).flatten(0, 1)
        inside = (pick >= 0) & (pick < 640)
        want = all_[pick.long().clamp(0, 639)] * inside[:, None, None]
        assert torch.equal(got[i].double(), want)         # products with powers of two: nothing is rounded
    e = cache.read(k, v, scales, pick[:0])
    assert e[0].shape == (0, 3, 128)


def test_scales_that_are_no_powers_of_two():
    """A cache from elsewhere: read and requantised with the same formulas."""
    gen = torch.Generator(device="cuda").manual_seed(18)
    k, v, scales = empty(3, 2, 16, 64, INT8)
    k.random_(-127, 128, generator=gen)
    scales.uniform_(0.01, 0.02, generator=gen)
    got, _ = cache.read(k, v, scales, torch.arange(48, dtype=torch.int32, device="cuda"))
    want = (k.float() * scales[..., :1, None]).half().transpose(1, 2).flatten(0, 1)
    assert torch.equal(got, want)
    before = k.double().clone() * scales[..., :1, None].double()
    x = rows(gen, 2, 4, 64, torch.float16) * 5
    cache.write(k, v, scales, x[:, :2], x[:, 2:], torch.tensor([21, 22], dtype=torch.int32, device="cuda"))
    after = k.double() * scales[..., :1, None].double()
    assert ((after - before)[1, :, :5].abs() <= 0.5001 * scales[1, :, :1, None].double()).all() and torch.equal(after[0], before[0])


def test_on_another_stream_after_work_on_it():
    gen = torch.Generator(device="cuda").manual_seed(11)
    k, v, scales = empty(40, 4, 16, 128, INT8)
    x, slots = rows(gen, 600, 8, 128, torch.float16), slots_of(16, 40, [(0, 600)], 1)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        y = x * 2
        for _ in range(30):
            y = y + x
        cache.write(k, v, scales, y[:, :4], y[:, 4:], slots)
        got = cache.read(k, v, scales, slots)
    stream.synchronize()
    k2, v2, s2 = empty(40, 4, 16, 128, INT8)
    cache.write(k2, v2, s2, y[:, :4], y[:, 4:], slots)
    want = cache.read(k2, v2, s2, slots)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(scales, s2)


def test_refusals():
    gen = torch.Generator(device="cuda").manual_seed(1)
    k, v, scales = empty(4, 2, 16, 64, INT8)
    x = rows(gen, 3, 4, 64, torch.float16)
    kk, vv, slots = x[:, :2], x[:, 2:], torch.arange(3, dtype=torch.int32, device="cuda")
    cache.write(k, v, scales, kk, vv, slots)
    cache.write(k, v, scales, kk[:0], vv[:0], slots[:0])
    bad_value = [(k.cpu(), v, scales, kk, vv, slots), (k, v[:3], scales, kk, vv, slots), (k, v, scales[:3], kk, vv, slots), (k, v, scales, kk.cpu(), vv, slots),
                 (k, v, scales, kk[:, :1], vv[:, :1], slots), (k, v, scales, kk[:2], vv, slots), (k, v, scales, kk, vv, slots[:2]),
                 (k, v, scales, kk, vv, slots[None]), (k, v, scales, kk[..., :32], vv[..., :32], slots), (k, v, scales.cpu(), kk, vv, slots),
                 (k.transpose(2, 3), v.transpose(2, 3), scales, kk, vv, slots), (k, v, scales, kk, vv, slots.cpu()), (k[0], v[0], scales, kk, vv, slots)]
    for args in bad_value:
        with pytest.raises(ValueError):
            cache.write(*args)
    bad_type = [(k.short(), v, scales, kk, vv, slots), (k, v.view(E4M3), scales, kk, vv, slots), (k, v, scales.half(), kk, vv, slots),
                (k, v, scales, kk.float(), vv, slots), (k, v, scales, kk, vv, slots.long())]
    for args in bad_type:
        with pytest.raises(TypeError):
            cache.write(*args)
    with pytest.raises(ValueError):
        cache.write(k, v, scales, kk, vv.bfloat16(), slots)
    with pytest.raises(TypeError):
        cache.read(k, v, scales, slots, torch.float32)

    def status(call):
        with pytest.raises(ops.Int4MatmulError) as e:
            call()
        return e.value.status
    odd = torch.zeros((3, 2, 4 * 64 + 4), dtype=torch.float16, device="cuda")[:, :, :64]
    assert status(lambda: cache.write(k, v, scales, odd, vv, slots)) == capi.ERR_ALIGN
    for shape in ((4, 2, 8, 64), (4, 2, 48, 64), (4, 2, 16, 96), (4, 2, 16, 32)):
        a, b, s = empty(*shape, INT8)
        y = torch.zeros((3, 2, shape[3]), dtype=torch.float16, device="cuda")
        assert status(lambda: cache.write(a, b, s, y, y, slots)) == capi.ERR_UNSUPPORTED
        assert status(lambda: cache.read(a, b, s, slots)) == capi.ERR_UNSUPPORTED
    wide = torch.zeros((4, 2, 16, 72), dtype=torch.int8, device="cuda")[..., :64]
    assert status(lambda: cache.read(wide, wide, scales, slots)) == capi.ERR_ALIGN
    assert MOST[INT8] == 127
