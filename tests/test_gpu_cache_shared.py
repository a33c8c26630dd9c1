"""GPU: attention of requests that share prefixes, against 64 bits and against requests that hold everything themselves."""
import math

import pytest
import torch

from cache_reference import attention_bound, values
from int4matmul_kernels_b200 import cache, capi, ops
from shared_reference import attention as reference
from test_gpu_cache_attention import BF16, E4M3, FP16, INT8, ints, make, queries

pytestmark = pytest.mark.gpu


def sums(v):
    out = [0]
    for n in v:
        out.append(out[-1] + n)
    return out


def check(q, k, v, scales, table, seq, lens, of, scale=None, window=0, max_len=None):
    """Both ways that the kernel for a request's own tokens is chosen: with the table as it is, and with one of so many places that it is not little work."""
    cu, seq = ints(sums(lens)), ints(seq)
    shared = cache.share(ints(of), seq, cu, q.shape[0])
    s = 1 / math.sqrt(q.shape[2]) if scale is None else scale
    out, size, reach, tail = reference(q, values(k, scales[..., 0]), values(v, scales[..., 1]), table, seq, cu, shared.prefix_of.tolist(), s, window)
    limit = attention_bound(out, size, reach, tail, q.dtype)
    wide = torch.full((table.shape[0], table.shape[1] + 200000 // k.shape[2]), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    results = []
    for t in (table, wide):
        got = cache.attention(q, k, v, scales, t, seq, cu, max(lens) if max_len is None else max_len, scale=scale, window=window, shared=shared)
        assert capi.load().i4mm_last_attention_kernels() & capi.ATTENTION_PREFIX
        assert got.shape == q.shape and got.dtype == q.dtype and got.is_contiguous()
        off = (got.double() - out).abs()
        assert (off <= limit).all(), ((off / limit).max().item(), (off > limit).nonzero()[:3].tolist())
        assert (got[(size == 0).all(-1)] == 0).all()
        results.append(got)
    return results[0]


@pytest.mark.parametrize("held,dtype", [(INT8, FP16), (INT8, BF16), (E4M3, FP16), (E4M3, BF16)])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_single_tokens(page, dim, held, dtype):
    """Prefixes of one token to a few thousand, odd ones and the edges of pages and tiles; readers with one token and more; a request without."""
    prefixes = [1, 2, 15, 16, 17, 31, 33, 127, 128, 129, 257, 1000, 2500]
    n = len(prefixes)
    own = [1 + (7 * i) % 40 for i in range(2 * n)] + [50]
    k, v, scales, table, gen = make(prefixes + own, 3, page, dim, held, page + dim)
    check(queries(gen, len(own), 3, dim, dtype), k, v, scales, table, prefixes + own, [0] * n + [1] * len(own), [-1] * n + [i % n for i in range(2 * n)] + [-1])


@pytest.mark.parametrize("readers", [1, 2, 7, 8, 9, 15, 16, 17, 31, 33, 63, 64, 65, 100, 127, 128, 129, 130, 200, 257, 300])
@pytest.mark.parametrize("heads,group", [(2, 1), (1, 8)])
def test_numbers_of_readers(readers, heads, group):
    own = [1 + i % 30 for i in range(readers)]
    for dim, held, dtype in ((128, INT8, FP16), (64, E4M3, BF16)):
        k, v, scales, table, gen = make([333] + own, heads, 16, dim, held, readers)
        check(queries(gen, readers, heads * group, dim, dtype), k, v, scales, table, [333] + own, [0] + [1] * readers, [-1] + [0] * readers)


@pytest.mark.parametrize("held", [INT8, E4M3])
@pytest.mark.parametrize("heads,group", [(1, 1), (1, 7), (2, 2), (8, 5), (40, 1), (2, 8), (3, 9), (1, 16), (2, 17), (1, 71)])
def test_head_layouts(heads, group, held):
    seqs, lens = [700, 70, 1, 333, 25], [0, 1, 1, 1, 1]
    for dim, dtype in ((128, FP16), (64, BF16)):
        k, v, scales, table, gen = make(seqs, heads, 16, dim, held, heads + group)
        check(queries(gen, 4, heads * group, dim, dtype), k, v, scales, table, seqs, lens, [-1, 0, 0, 0, 0])


@pytest.mark.parametrize("order", ["heads", "tokens"])
@pytest.mark.parametrize("prefix,readers,heads", [(40000, 3, 4), (20000, 40, 1), (5000, 150, 2), (900, 5, 40), (130, 400, 4), (128, 30, 30)])
def test_work_over_the_whole_gpu(prefix, readers, heads, order):
    """Long and short prefixes under few and many heads: cut over blocks, many in one block."""
    own = [1 + i % 9 for i in range(readers)]
    k, v, scales, table, gen = make([prefix] + own, heads, 32, 128, INT8, prefix + readers, order)
    check(queries(gen, readers, 2 * heads, 128, FP16), k, v, scales, table, [prefix] + own, [0] + [1] * readers, [-1] + [0] * readers)


@pytest.mark.parametrize("held,dtype", [(INT8, FP16), (E4M3, BF16)])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,group", [(2, 1), (2, 4), (1, 8)])
def test_drafts_and_chunks(heads, group, dim, held, dtype):
    """Several rows a request, one of them a chunk that the other kernel takes; prefixes in the middle of the batch, one of them growing itself."""
    lens = [3, 0, 1, 4, 300, 8, 0, 2, 60, 1]
    seqs = [7, 450, 30, 4, 320, 100, 1300, 2, 60, 900]
    of = [1, -1, 6, 6, 1, -1, -1, 6, -1, 8]
    k, v, scales, table, gen = make(seqs, heads, 16, dim, held, group)
    check(queries(gen, sum(lens), heads * group, dim, dtype), k, v, scales, table, seqs, lens, of)


@pytest.mark.parametrize("window", [1, 5, 30, 100, 128, 333, 5000])
def test_windows(window):
    """Counted over prefix and own tokens; some hide the whole prefix from some rows."""
    lens, seqs, of = [0, 1, 1, 3, 100, 1], [400, 1, 40, 90, 130, 700], [-1, 0, 0, 0, 0, 0]
    for group, dim in ((1, 128), (4, 64)):
        k, v, scales, table, gen = make(seqs, 2, 32, dim, INT8, window)
        check(queries(gen, sum(lens), 2 * group, dim, FP16), k, v, scales, table, seqs, lens, of, window=window)


@pytest.mark.parametrize("scale", [0.0, -0.1, 0.5, 3.0])
def test_scales(scale):
    seqs, lens = [600, 3, 44, 20], [0, 1, 2, 1]
    for held, dtype in ((INT8, FP16), (E4M3, BF16)):
        k, v, scales, table, gen = make(seqs, 2, 16, 128, held, 9)
        check(queries(gen, 4, 4, 128, dtype, 0.3), k, v, scales, table, seqs, lens, [-1, 0, 0, 0], scale=scale)


def test_steep_rows():
    """The largest score comes late, again and again, in the prefix and then in a request's own tokens, or stays in the first tile."""
    for rising in (True, False):
        seqs, lens = [1500, 100, 30], [0, 1, 1]
        k, v, scales, table, gen = make(seqs, 2, 16, 128, INT8, 3, spread=0)
        scales.fill_(2.0 ** -4)
        length = torch.arange(1500, device="cuda") * (1 if rising else -1) + (0 if rising else 1500)
        for i in range(1500):
            k[table[0, i // 16].long(), :, i % 16] = (length[i] // 12).clamp(max=127).to(INT8)
        q = torch.full((2, 4, 128), 0.5, device="cuda").half()
        check(q, k, v, scales, table, seqs, lens, [-1, 0, 0])


def test_missing_and_unused_pages():
    """Pages that there are not hide their tokens; what lies behind the last token of a page, in scales too, is of no account."""
    seqs, lens = [300, 20, 33], [0, 1, 2]
    for held in (INT8, E4M3):
        k, v, scales, table, gen = make(seqs, 2, 16, 64, held, 4)
        table[0, 3] = -1
        table[0, 7] = 10 ** 6
        table[1, 0] = -1
        if held == E4M3:
            last = table[0, 300 // 16].long()
            for c in (k, v):
                c.view(INT8)[last, :, 300 % 16:] = 0x7F                       # NaN
        check(queries(gen, 3, 4, 64, FP16), k, v, scales, table, seqs, lens, [-1, 0, 0])
    table[0] = -1                                                             # nothing of the prefix is there
    check(queries(gen, 3, 4, 64, FP16), k, v, scales, table, seqs, lens, [-1, 0, 0])


def test_rows_without_tokens_and_padding():
    """Requests with more rows than tokens, rows behind the last request, a prefix longer than its row of the table."""
    k, v, scales, table, gen = make([100, 0, 2, 9], 2, 16, 64, INT8, 6)
    seqs, lens = [100, 0, 2, 9], [0, 2, 5, 1]
    q = queries(gen, 11, 4, 64, BF16)
    got = check(q, k, v, scales, table, seqs, lens, [-1, 0, 0, 0])
    assert (got[:5] == 0).all() and (got[5:8] != 0).any() and (got[8:] == 0).all()
    check(q, k, v, scales, table, [5000, 0, 2, 9], lens, [-1, 0, 0, 0])


def test_equal_to_requests_that_hold_everything():
    """The same tokens held by every request: nothing but the order of the sums differs."""
    seqs, lens = [512, 60, 7, 130], [0, 1, 4, 2]
    k, v, scales, table, gen = make(seqs, 4, 16, 128, INT8, 8)
    q = queries(gen, 7, 8, 128, FP16)
    got = check(q, k, v, scales, table, seqs, lens, [-1, 0, 0, 0])
    whole = torch.cat([table[:1, :32].expand(4, -1), table], 1).contiguous()
    other = cache.attention(q, k, v, scales, whole, ints([512, 572, 519, 642]), ints(sums(lens)), 4)
    assert (got.float() - other.float()).abs().max() < 2e-3 * other.float().abs().max()


@pytest.mark.parametrize("window", [0, 90, 20000])
@pytest.mark.parametrize("held,dtype,dim", [(INT8, BF16, 128), (E4M3, FP16, 64)])
def test_parts_of_a_prefix_under_rows_of_chunks(held, dtype, dim, window):
    """One head of a long prefix: all blocks have a part, and rows of a chunk, of drafts and of single tokens add them up."""
    seqs, lens, of = [30000, 130, 1, 50, 6], [0, 101, 1, 4, 1], [-1, 0, 0, 0, 0]
    k, v, scales, table, gen = make(seqs, 1, 64, dim, held, window)
    check(queries(gen, sum(lens), 2, dim, dtype), k, v, scales, table, seqs, lens, of, window=window)


@pytest.mark.parametrize("readers", [255, 256, 257])
def test_rows_that_both_kernels_take(readers):
    """Places on both sides of what the kernel of few readers takes, in one call, and more places than a warp keeps in registers."""
    prefixes = [300, 70] + [20 + i for i in range(40)]
    of = [-1] * 42 + [0] * readers + [1] * 40 + [2 + i for i in range(40)]
    own = [1 + i % 5 for i in range(readers + 80)]
    k, v, scales, table, gen = make(prefixes + own, 2, 16, 64, INT8, readers)
    check(queries(gen, len(own), 2, 64, FP16), k, v, scales, table, prefixes + own, [0] * 42 + [1] * len(own), of)


def test_which_kernels_run():
    seqs, lens = [100] + [3] * 257, [0] + [1] * 257
    k, v, scales, table, gen = make(seqs, 1, 16, 64, INT8, 1)
    for readers, many in ((1, False), (256, False), (257, True)):
        seq, cu = ints(seqs[:readers + 1]), ints(sums(lens[:readers + 1]))
        shared = cache.share(ints([-1] + [0] * readers), seq, cu, readers)
        cache.attention(queries(gen, readers, 1, 64, FP16), k, v, scales, table[:readers + 1], seq, cu, 1, shared=shared)
        ran = capi.load().i4mm_last_attention_kernels()
        assert ran & capi.ATTENTION_PREFIX and ran & capi.ATTENTION_FEW_ROWS and bool(ran & capi.ATTENTION_MANY_READERS) == many


def test_no_requests():
    k, v, scales, table, gen = make([20], 2, 16, 64, INT8, 1)
    q = queries(gen, 3, 2, 64, FP16)
    shared = cache.share(ints([]), ints([]), ints([0]), 3)
    assert shared.rows.tolist() == [-1] * 3 and shared.positions.tolist() == [-1] * 3
    got = cache.attention(q, k, v, scales, table[:0], ints([]), ints([0]), 1, shared=shared)
    assert (got == 0).all() and not capi.load().i4mm_last_attention_kernels() & capi.ATTENTION_PREFIX


def test_nobody_shares():
    """Tables without a reader: a call without them, but for the order of fp32 operations, which may differ from one compiled kernel to the other.  So
    both results are fp16 roundings of numbers that are 2^-17 of the summands apart at most, and so one step (2^-10) apart at most, and that."""
    seqs, lens = [100, 300, 2000], [1, 2, 1]
    k, v, scales, table, gen = make(seqs, 2, 16, 128, INT8, 8)
    q, cu = queries(gen, 4, 8, 128, FP16), ints(sums(lens))
    a = check(q, k, v, scales, table, seqs, lens, [-1, -1, 7]).double()
    b = cache.attention(q, k, v, scales, table, ints(seqs), cu, 2).double()
    size = reference(q, values(k, scales[..., 0]), values(v, scales[..., 1]), table, ints(seqs), cu, [-1] * 3, 128 ** -0.5)[1]
    assert ((a - b).abs() <= a.abs() * 2.0 ** -10 + size * 2.0 ** -17 + 2.0 ** -24).all()


def test_infinite_queries_stay_in_their_rows():
    seqs, lens = [200, 10, 10, 10], [0, 1, 1, 1]
    k, v, scales, table, gen = make(seqs, 2, 16, 128, INT8, 2)
    q = queries(gen, 3, 2, 128, FP16)
    want = check(q, k, v, scales, table, seqs, lens, [-1, 0, 0, 0])
    q[1, 0, 3], q[1, 1, 4] = float("nan"), float("inf")
    shared = cache.share(ints([-1, 0, 0, 0]), ints(seqs), ints(sums(lens)), 3)
    got = cache.attention(q, k, v, scales, table, ints(seqs), ints(sums(lens)), 1, shared=shared)
    assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2]) and got[1].isnan().all()


def test_the_same_bits_again_on_any_stream_and_in_a_graph():
    seqs, lens, of = [3000] + [20 + i for i in range(50)], [0] + [1] * 50, [-1] + [0] * 50
    k, v, scales, table, gen = make(seqs, 8, 16, 128, INT8, 5)
    q, seq, cu = queries(gen, 50, 16, 128, FP16), ints(seqs), ints(sums(lens))
    shared = cache.share(ints(of), seq, cu, 50)
    call = lambda: cache.attention(q, k, v, scales, table, seq, cu, 1, shared=shared)  # noqa: E731
    want = call()
    for _ in range(20):
        assert torch.equal(call(), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    got.zero_()
    for _ in range(3):
        graph.replay()
    assert torch.equal(got, want)
    # a replay goes by what the tables hold then
    seq[0] = 1000
    for a, b in zip(shared, cache.share(ints(of), seq, cu, 50)):
        a.copy_(b)
    graph.replay()
    assert torch.equal(got, call()) and not torch.equal(got, want)
    ops.check_device_status()


def test_calls_of_two_streams_at_once():
    seqs, lens, of = [2000] + [30] * 20, [0] + [1] * 20, [-1] + [0] * 20
    k, v, scales, table, gen = make(seqs, 8, 16, 128, INT8, 5)
    qs, seq, cu = [queries(gen, 20, 8, 128, FP16) for _ in range(2)], ints(seqs), ints(sums(lens))
    shared = cache.share(ints(of), seq, cu, 20)
    want = [cache.attention(q, k, v, scales, table, seq, cu, 1, shared=shared) for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    got = []
    for _ in range(30):
        for q, stream in zip(qs, streams):
            with torch.cuda.stream(stream):
                got.append(cache.attention(q, k, v, scales, table, seq, cu, 1, shared=shared))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i % 2]) for i, g in enumerate(got))


def test_without_cu_lens():
    seqs = [1, 200, 30]
    k, v, scales, table, gen = make(seqs, 2, 16, 64, INT8, 7)
    q = queries(gen, 3, 2, 64, FP16)
    shared = cache.share(ints([1, -1, 1]), ints(seqs), ints([0, 1, 2, 3]), 3)
    a = cache.attention(q, k, v, scales, table, ints(seqs), shared=shared)
    assert torch.equal(a, cache.attention(q, k, v, scales, table, ints(seqs), ints([0, 1, 2, 3]), 1, shared=shared))


def test_offsets_beyond_32_bits():
    """A cache of more than 4 GB of which the last pages are used."""
    pages, heads, page = 2 ** 32 // (8 * 128 * 128) + 64, 8, 128
    k, v = (torch.zeros((pages, heads, page, 128), dtype=INT8, device="cuda") for _ in range(2))
    scales = torch.full((pages, heads, 2), 2.0 ** -6, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(1)
    for c in (k, v):
        c[-40:] = torch.randint(-127, 128, (40, heads, page, 128), dtype=INT8, device="cuda", generator=gen)
    table = torch.arange(pages - 40, pages - 40 + 32, dtype=torch.int32, device="cuda").view(2, 16).contiguous()
    seqs, lens = [16 * 128 - 3, 130], [0, 1]
    cu, seq, q = ints(sums(lens)), ints(seqs), queries(gen, 1, 8, 128, FP16)
    shared = cache.share(ints([-1, 0]), seq, cu, 1)
    got = cache.attention(q, k, v, scales, table, seq, cu, 1, shared=shared)
    small = torch.arange(32, dtype=torch.int32, device="cuda").view(2, 16)
    last = [t[-40:-8].contiguous() for t in (k, v, scales)]
    assert torch.equal(got, cache.attention(q, *last, small, seq, cu, 1, shared=shared))


def test_tables_of_anything_stay_within_bounds():
    """Lists that no call of share makes are wrong answers, but nothing beyond the arrays is read or written."""
    seqs, lens = [200, 10, 10, 10], [0, 1, 1, 1]
    k, v, scales, table, gen = make(seqs, 2, 16, 128, INT8, 2)
    q, seq, cu = queries(gen, 3, 2, 128, FP16), ints(seqs), ints(sums(lens))
    of = ints([-1, 0, 0, 0])
    for starts, rows in (([0, 9, 9, 9, 9], [0, 1, 2]), ([5, -3, 2, 1, 3], [0, 1, 2]), ([0, 3, 3, 3, 3], [7, -1, 10 ** 9]), ([0] * 5, [0, 1, 2])):
        got = cache.attention(q, k, v, scales, table, seq, cu, 1, shared=cache.Shared(of, ints(starts), ints(rows), ints([0, 0, 0])))
        assert got.shape == q.shape
    torch.cuda.synchronize()
    check(q, k, v, scales, table, seqs, lens, [-1, 0, 0, 0])


def test_refusals():
    seqs, lens = [200, 10], [0, 1]
    k, v, scales, table, gen = make(seqs, 2, 16, 128, INT8, 2)
    q, seq, cu = queries(gen, 1, 2, 128, FP16), ints(seqs), ints(sums(lens))
    good = cache.share(ints([-1, 0]), seq, cu, 4)
    for error, bad in ((ValueError, dict(prefix_of=ints([-1]))), (ValueError, dict(starts=ints([0, 1]))), (ValueError, dict(rows=ints([]))),
                       (TypeError, dict(rows=good.rows.long())), (ValueError, dict(prefix_of=good.prefix_of.cpu())), (ValueError, dict(rows=ints([[0]])))):
        with pytest.raises(error):
            cache.attention(q, k, v, scales, table, seq, cu, 1, shared=good._replace(**bad))
