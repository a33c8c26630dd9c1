"""GPU: attention over the paged 8-bit cache against 64 bits."""
import math

import pytest
import torch

from cache_reference import attention as reference, attention_bound, values
from int4matmul_kernels_b200 import cache, capi, ops

pytestmark = pytest.mark.gpu
INT8, E4M3 = torch.int8, torch.float8_e4m3fn
FP16, BF16 = torch.float16, torch.bfloat16


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def make(seqs, heads, page, dim, held, seed, order="heads", spread=0.7, spare=3):
    """A filled cache and the block table of requests of these lengths; every place that no token has holds the largest bytes."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    counts = [-(-s // page) for s in seqs]
    pages, width = sum(counts) + spare, max([1] + counts)
    shape = (pages, page, heads, dim) if order == "tokens" else (pages, heads, page, dim)
    arrays = []
    for _ in range(2):
        c = torch.randint(-127, 128, shape, dtype=torch.int8, device="cuda", generator=gen)
        if held == E4M3:                                    # any byte but NaN, fewer of the large ones
            c = ((torch.randn(shape, device="cuda", generator=gen) * 40).clamp(-448, 448)).to(E4M3).view(INT8)
        arrays.append((c.transpose(1, 2) if order == "tokens" else c).view(held))
    scales = torch.exp2(torch.randint(-8, -4, (pages, heads, 2), device="cuda", generator=gen).float())
    if spread:
        scales = scales * torch.exp(spread * torch.randn(scales.shape, device="cuda", generator=gen))
    perm = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(seqs), width), -1, dtype=torch.int32)
    for b, (n, s) in enumerate(zip(counts, seqs)):
        ids = [perm.pop() for _ in range(n)]
        table[b, :n] = torch.tensor(ids, dtype=torch.int32)
        if s % page:
            for c in arrays:
                c.view(INT8)[ids[-1], :, s % page:] = 126
    return arrays[0], arrays[1], scales, table.cuda(), gen


def check(q, k, v, scales, table, seq, cu=None, max_len=1, scale=None, window=0):
    got = cache.attention(q, k, v, scales, table, seq, cu, max_len, scale=scale, window=window)
    assert got.shape == q.shape and got.dtype == q.dtype and got.is_contiguous()
    # The kernel is chosen by how much work a call may be, which the table's width bounds: one with many places for pages that are not there is
    # more, and takes the prompt kernel for requests of more than 64 rows.
    wide = torch.full((table.shape[0], table.shape[1] + 200000 // k.shape[2]), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    other = cache.attention(q, k, v, scales, wide, seq, cu, max_len, scale=scale, window=window)
    s = 1 / math.sqrt(q.shape[2]) if scale is None else scale
    out, size, reach, tail = reference(q, values(k, scales[..., 0]), values(v, scales[..., 1]), table, seq, cu, s, window)
    limit = attention_bound(out, size, reach, tail, q.dtype)
    for result in (got, other):
        off = (result.double() - out).abs()
        assert (off <= limit).all(), ((off / limit).max().item(), (off > limit).nonzero()[:3].tolist())
        assert (result[(size == 0).all(-1)] == 0).all()
    return got


def queries(gen, tokens, heads, dim, dtype, size=1.0):
    return (torch.randn((tokens, heads, dim), device="cuda", generator=gen) * size).to(dtype)


@pytest.mark.parametrize("held,dtype", [(INT8, FP16), (INT8, BF16), (E4M3, FP16), (E4M3, BF16)])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_single_tokens(page, dim, held, dtype):
    """Lengths from none and one to a few thousand, odd ones and the edges of pages and tiles."""
    seqs = [1, 0, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 255, 257, 1000, 2500]
    k, v, scales, table, gen = make(seqs, 3, page, dim, held, page + dim)
    check(queries(gen, len(seqs), 3, dim, dtype), k, v, scales, table, ints(seqs))


@pytest.mark.parametrize("held", [INT8, E4M3])
@pytest.mark.parametrize("heads,group", [(1, 1), (1, 7), (2, 2), (8, 5), (40, 1), (2, 8), (3, 9), (1, 16), (2, 17), (1, 32), (1, 71)])
def test_head_layouts(heads, group, held):
    seqs = [70, 1, 333, 0, 1025]
    for dim, dtype in ((128, FP16), (64, BF16)):
        k, v, scales, table, gen = make(seqs, heads, 16, dim, held, heads + group)
        check(queries(gen, len(seqs), heads * group, dim, dtype), k, v, scales, table, ints(seqs))


@pytest.mark.parametrize("order", ["heads", "tokens"])
@pytest.mark.parametrize("b,length", [(1, 1), (1, 16), (1, 100), (1, 5000), (1, 40000), (200, 30), (300, 1), (37, 900)])
def test_work_over_the_whole_gpu(b, length, order):
    """Few and many requests, short and long: lengths cut over blocks, many of them in one block."""
    seqs = [max(1, length - 7 * (i % 5)) for i in range(b)]
    k, v, scales, table, gen = make(seqs, 4, 32, 128, INT8, b + length, order)
    check(queries(gen, b, 8, 128, FP16), k, v, scales, table, ints(seqs))


@pytest.mark.parametrize("held,dtype", [(INT8, FP16), (E4M3, BF16)])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,group", [(2, 1), (1, 3), (2, 4), (1, 8)])
def test_a_few_tokens_of_each_request(heads, group, dim, held, dtype):
    lens = [1, 2, 3, 4, 5, 8, 0, 1, 7, 9]
    seqs = [1, 2, 50, 64, 300, 8, 0, 1, 700, 1200]
    k, v, scales, table, gen = make(seqs, heads, 16, dim, held, group)
    cu = ints([0] + torch.tensor(lens).cumsum(0).tolist())
    check(queries(gen, sum(lens), heads * group, dim, dtype), k, v, scales, table, ints(seqs), cu, max(lens))


@pytest.mark.parametrize("held,dtype", [(INT8, FP16), (INT8, BF16), (E4M3, FP16), (E4M3, BF16)])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_prompts(page, dim, held, dtype):
    lens = [17, 130, 1, 300, 64]
    seqs = [17, 700, 90, 300, 65]
    k, v, scales, table, gen = make(seqs, 2, page, dim, held, page + 7 * dim)
    cu = ints([0] + torch.tensor(lens).cumsum(0).tolist())
    check(queries(gen, sum(lens), 4, dim, dtype), k, v, scales, table, ints(seqs), cu, max(lens))


@pytest.mark.parametrize("heads,group", [(1, 1), (5, 1), (1, 5), (2, 8), (1, 12), (1, 33), (1, 128), (1, 200)])
@pytest.mark.parametrize("length,before", [(128, 0), (129, 0), (257, 1000), (31, 3000), (600, 13)])
def test_prompt_lengths_and_groups(length, before, heads, group):
    k, v, scales, table, gen = make([before + length], heads, 16, 128, INT8, length + group)
    check(queries(gen, length, heads * group, 128, FP16), k, v, scales, table, ints([before + length]), ints([0, length]), length)


@pytest.mark.parametrize("window", [1, 5, 16, 100, 128, 129, 1000, 100000])
@pytest.mark.parametrize("lens", [[1] * 6, [3, 1, 4, 2, 8, 1], [200, 1, 17, 129, 40, 64]])
def test_windows(window, lens):
    seqs = [300, 1, 1500, 129, 64, 777]
    seqs = [max(s, n) for s, n in zip(seqs, lens)]
    for heads, group, dim in ((2, 2, 128), (1, 4, 64)):
        k, v, scales, table, gen = make(seqs, heads, 16, dim, INT8, window)
        cu = ints([0] + torch.tensor(lens).cumsum(0).tolist())
        check(queries(gen, sum(lens), heads * group, dim, FP16), k, v, scales, table, ints(seqs), cu, max(lens), window=window)


@pytest.mark.parametrize("lens", [[1] * 5, [2, 3, 1, 4, 1], [40, 3, 150, 1, 20]])
def test_rows_that_see_nothing(lens):
    """Requests of no tokens, rows before a request's first token, pages that are not there, rows of no request."""
    seqs = [0, max(0, lens[1] - 2), 200, 900, 33]
    k, v, scales, table, gen = make(seqs, 2, 16, 128, INT8, 5)
    table[3, 3] = -1
    table[3, 10:30] = 2 ** 30
    table[4, :] = -5
    cu = ints([0] + torch.tensor(lens).cumsum(0).tolist())
    q = queries(gen, sum(lens) + 9, 6, 128, FP16)
    got = check(q, k, v, scales, table, ints(seqs), cu, max(lens))
    assert (got[sum(lens):] == 0).all() and (got[:lens[0]] == 0).all() and (got[sum(lens) - lens[4]:] == 0).all()
    if max(lens) == 1:
        got = check(q, k, v, scales, table, ints(seqs), None, 1)
        assert (got[5:] == 0).all()


def test_lengths_beyond_the_table_and_no_requests():
    k, v, scales, table, gen = make([40, 64], 1, 16, 64, INT8, 6)
    check(queries(gen, 2, 2, 64, FP16), k, v, scales, table, ints([500, 2 ** 31 - 1]))
    check(queries(gen, 60, 2, 64, FP16), k, v, scales, table, ints([70, 64]), ints([0, 40, 60]), 40)
    got = cache.attention(queries(gen, 5, 2, 64, FP16), k, v, scales, table[:0], ints([]))
    assert (got == 0).all()
    got = cache.attention(queries(gen, 5, 2, 64, FP16), k, v, scales, table[:, :0], ints([3, 3]), ints([0, 2, 5]), 3)
    assert (got == 0).all()
    assert cache.attention(queries(gen, 0, 2, 64, FP16), k, v, scales, table, ints([3, 3]), ints([0, 0, 0]), 3).shape == (0, 2, 64)


@pytest.mark.parametrize("max_len", [0, 1, 64, 10 ** 6])
def test_a_wrong_max_len_changes_nothing_but_time(max_len):
    lens, seqs = [1, 150, 4, 1, 33], [600, 700, 4, 1, 90]
    k, v, scales, table, gen = make(seqs, 2, 16, 128, INT8, 61)
    cu = ints([0] + torch.tensor(lens).cumsum(0).tolist())
    check(queries(gen, sum(lens), 6, 128, FP16), k, v, scales, table, ints(seqs), cu, max_len)


@pytest.mark.parametrize("places", [0, 10000])
@pytest.mark.parametrize("lens", [[1, 1, 1], [3, 2, 1], [60, 1, 200]])
def test_bytes_and_scales_of_places_that_no_row_sees(lens, places):
    """The rest of a last page, and whole pages beyond it: NaN bytes, scales that are infinite or NaN."""
    seqs = [77, 201, 203]
    k, v, scales, table, gen = make(seqs, 2, 16, 128, E4M3, 62)
    table = torch.cat([table, torch.full((3, places), -1, dtype=torch.int32, device="cuda")], dim=1)
    cu = ints([0] + torch.tensor(lens).cumsum(0).tolist())
    q = queries(gen, sum(lens), 4, 128, BF16)
    want = check(q, k, v, scales, table, ints(seqs), cu, max(lens))
    used = torch.zeros(k.shape[0], dtype=torch.bool)
    for b, s in enumerate(seqs):
        ids = table[b, :-(-s // 16)].long().cpu()
        used[ids] = True
        if s % 16:
            k.view(INT8)[ids[-1], :, s % 16:] = 0x7F
            v.view(INT8)[ids[-1], :, s % 16:] = 0x7F
    k.view(INT8)[~used.cuda()] = 0x7F
    v.view(INT8)[~used.cuda()] = 0x7F
    scales[~used.cuda()] = math.nan
    assert torch.equal(cache.attention(q, k, v, scales, table, ints(seqs), cu, max(lens)), want)


@pytest.mark.parametrize("lens", [[1] * 4, [2, 5, 1, 3], [100, 40, 20, 300]])
@pytest.mark.parametrize("dtype", [FP16, BF16])
def test_sharp_and_flat_weights_and_scales_far_apart(lens, dtype):
    """Scores of hundreds, of next to nothing, and pages whose values are 2^20 times another's."""
    seqs = [400, 800, 30, 300]
    cu = ints([0] + torch.tensor(lens).cumsum(0).tolist())
    for size in (30.0, 1e-4):
        k, v, scales, table, gen = make(seqs, 2, 16, 128, INT8, 63)
        check(queries(gen, sum(lens), 2, 128, dtype, size), k, v, scales, table, ints(seqs), cu, max(lens))
    k, v, scales, table, gen = make(seqs, 2, 16, 128, INT8, 64)
    scales[..., 1] *= torch.exp2(torch.randint(-10, 11, scales.shape[:2], device="cuda", generator=gen).float())
    q = queries(gen, sum(lens), 2, 128, dtype)
    got = cache.attention(q, k, v, scales, table, ints(seqs), cu, max(lens))
    assert torch.isfinite(got).all() or dtype == FP16
    check(q * 0.3, k, v, scales * 2.0 ** -6, table, ints(seqs), cu, max(lens))


def test_queries_of_extreme_size():
    """bf16 queries far outside of fp16's range, against scales that bring the scores back."""
    seqs = [300, 90]
    for size in (2.0 ** 60, 2.0 ** -60):
        for lens in ([1, 1], [30, 90]):
            k, v, scales, table, gen = make(seqs, 1, 16, 128, INT8, 65)
            cu = ints([0, lens[0], sum(lens)])
            check(queries(gen, sum(lens), 2, 128, BF16, size), k, v, scales, table, ints(seqs), cu, max(lens), scale=1 / (size * 11.3))


def test_query_strides():
    seqs, lens = [100, 40, 300], [1, 3, 40]
    k, v, scales, table, gen = make(seqs, 2, 16, 64, INT8, 66)
    cu = ints([0, 1, 4, 44])
    wide = queries(gen, 44, 12, 64, FP16)
    q = wide[:, 2:6]
    assert torch.equal(check(q, k, v, scales, table, ints(seqs), cu, 40), cache.attention(q.contiguous(), k, v, scales, table, ints(seqs), cu, 40))
    q = queries(gen, 4, 44, 64, FP16).transpose(0, 1)
    check(q, k, v, scales, table, ints(seqs), cu, 40)
    padded = torch.full((3, table.shape[1] + 5), 7, dtype=torch.int32, device="cuda")
    padded[:, 2:2 + table.shape[1]] = table
    check(q, k, v, scales, padded[:, 2:2 + table.shape[1]], ints(seqs), cu, 40)


def test_a_cache_whose_offsets_pass_32_bits():
    """4.3 GB of keys: the last pages lie beyond 2^32 bytes."""
    heads, page, dim = 8, 128, 128
    pages = (2 ** 32) // (heads * page * dim) + 40
    k = torch.zeros((pages, heads, page, dim), dtype=INT8, device="cuda")
    v = torch.zeros((pages, heads, page, dim), dtype=INT8, device="cuda")
    scales = torch.full((pages, heads, 2), 2.0 ** -6, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(2)
    x = queries(gen, 400, 2 * heads, dim, FP16)
    ids = [pages - 1, 3, pages - 30, pages - 2]
    slots = ints([ids[p // page] * page + p % page for p in range(400)])
    cache.write(k, v, scales, x[:, :heads], x[:, heads:], slots)
    table, sub = ints([ids]), torch.tensor(ids, device="cuda")
    kk, vv, ss = k[sub].clone(), v[sub].clone(), scales[sub].clone()
    for lens in (1, 300):
        q, cu = queries(gen, lens, heads, dim, FP16), ints([0, lens])
        got = cache.attention(q, k, v, scales, table, ints([400]), cu, lens)
        assert torch.equal(got, cache.attention(q, kk, vv, ss, ints([[0, 1, 2, 3]]), ints([400]), cu, lens))
    r = cache.read(k, v, scales, slots)
    assert (r[0] - x[:, :heads]).abs().max() < 0.05 and r[0].abs().max() > 1


@pytest.mark.parametrize("places", [0, 10000])
@pytest.mark.parametrize("lens", [[1] * 30, [2] * 30, [90] + [1] * 28 + [200]])
def test_repeated_calls_give_the_same_bits(lens, places):
    """Beside other work on another stream too: nothing depends on which block comes first."""
    seqs = [max(n, 37 * (i + 3) % 4000) for i, n in enumerate(lens)]
    k, v, scales, table, gen = make(seqs, 4, 16, 128, INT8, 67)
    table = torch.cat([table, torch.full((len(seqs), places), -1, dtype=torch.int32, device="cuda")], dim=1)
    cu = ints([0] + torch.tensor(lens).cumsum(0).tolist())
    q = queries(gen, sum(lens), 8, 128, FP16)
    first = cache.attention(q, k, v, scales, table, ints(seqs), cu, max(lens))
    other = torch.cuda.Stream()
    a = torch.randn((4096, 4096), device="cuda")
    torch.cuda.synchronize()
    for i in range(10):
        with torch.cuda.stream(other):
            b = a @ a
        assert torch.equal(cache.attention(q, k, v, scales, table, ints(seqs), cu, max(lens)), first)
    del b


def test_on_another_stream_and_in_a_graph():
    seqs = [500, 30, 2000]
    k, v, scales, table, gen = make(seqs, 4, 16, 128, INT8, 68)
    q, seq = queries(gen, 3, 8, 128, FP16), ints(seqs)
    want = cache.attention(q, k, v, scales, table, seq)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        x = q * 0
        for _ in range(20):
            x = x + q / 16
        y = x - q * 0.25
        got = cache.attention(y, k, v, scales, table, seq)
        same = cache.attention(y.clone(), k, v, scales, table, seq)
    stream.synchronize()
    assert torch.equal(got, same)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache.attention(q, k, v, scales, table, seq)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    seq.copy_(ints([499, 1, 1700]))                             # a captured call follows the lengths on the GPU
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, cache.attention(q, k, v, scales, table, seq))


def test_refusals():
    k, v, scales, table, gen = make([40, 40], 2, 16, 64, INT8, 69)
    q, seq, cu = queries(gen, 2, 4, 64, FP16), ints([40, 40]), ints([0, 1, 2])
    cache.attention(q, k, v, scales, table, seq, cu)
    for args in ((q.cpu(), k, v, scales, table, seq, cu), (q[:, :3], k, v, scales, table, seq, cu), (q[..., :32], k, v, scales, table, seq, cu),
                 (q, k, v, scales, table, seq[:1], cu), (q, k, v, scales, table, seq, cu[:2]), (q, k, v, scales, table[0], seq, cu),
                 (q, k, v, scales, table, seq.cpu(), cu), (q[:1], k, v, scales, table, seq), (q, k, v, scales, table.t(), seq, cu),
                 (q[0], k, v, scales, table, seq, cu), (q, k, v, scales, table, seq, cu, -1)):
        with pytest.raises(ValueError):
            cache.attention(*args)
    with pytest.raises(ValueError):
        cache.attention(q, k, v, scales, table, seq, cu, window=-1)
    for args in ((q.float(), k, v, scales, table, seq, cu), (q, k, v, scales, table.long(), seq, cu), (q, k, v, scales, table, seq.long(), cu),
                 (q, k, v, scales, table, seq, cu.long())):
        with pytest.raises(TypeError):
            cache.attention(*args)
    odd = torch.zeros((2, 4, 68), dtype=FP16, device="cuda")[..., :64]
    with pytest.raises(ops.Int4MatmulError) as e:
        cache.attention(odd, k, v, scales, table, seq, cu)
    assert e.value.status == capi.ERR_ALIGN
