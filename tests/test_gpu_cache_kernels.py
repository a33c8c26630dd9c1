"""GPU: which kernels an attention call launched, and the prompt kernel on windows, scales and offsets that the rule for little work would keep from it."""
import math

import pytest
import torch

from cache_reference import attention as reference, attention_bound, values
from int4matmul_kernels_b200 import cache, capi
from test_gpu_cache_attention import BF16, E4M3, FP16, INT8, ints, make, queries

pytestmark = pytest.mark.gpu
FEW, PROMPT, BOTH = capi.ATTENTION_FEW_ROWS, capi.ATTENTION_PROMPT, capi.ATTENTION_FEW_ROWS | capi.ATTENTION_PROMPT


def run(kernels, q, k, v, scales, table, seq, cu=None, max_len=1, scale=None, window=0):
    """The output, which is within its bound of 64 bits; asserts which kernels gave it."""
    got = cache.attention(q, k, v, scales, table, seq, cu, max_len, scale=scale, window=window)
    assert capi.load().i4mm_last_attention_kernels() == kernels
    s = 1 / math.sqrt(q.shape[2]) if scale is None else scale
    kk, vv = values(k, scales[..., 0]), values(v, scales[..., 1])
    out, size, _, tail = reference(q, kk, vv, table, seq, cu, s, window)
    reach = reference(q, kk, vv, table, seq, cu, abs(s), window)[2]              # (a bound on |scores|: the sign does not matter to it)
    limit = attention_bound(out, size, reach, tail, q.dtype)
    off = (got.double() - out).abs()
    assert (off <= limit).all(), ((off / limit).max().item(), (off > limit).nonzero()[:3].tolist())
    assert (got[(size == 0).all(-1)] == 0).all()
    return got


def wide(table, page, places=200000):
    """The table with room for many more tokens: more work for all that the rule knows."""
    out = torch.full((table.shape[0], table.shape[1] + places // page), -1, dtype=torch.int32, device="cuda")
    out[:, :table.shape[1]] = table
    return out


def packed(lens):
    return ints([0] + torch.tensor(lens).cumsum(0).tolist())


def test_which_kernels_run():
    k, v, scales, table, gen = make([300, 40], 2, 16, 64, INT8, 1)
    seq, cu = ints([300, 40]), packed([200, 1])
    q = queries(gen, 201, 4, 64, FP16)
    run(FEW, q[:2], k, v, scales, table, seq)
    run(FEW, q, k, v, scales, table, seq, cu, 200)                               # little work
    run(BOTH, q, k, v, scales, wide(table, 16), seq, cu, 200)
    run(FEW, q, k, v, scales, wide(table, 16), seq, cu, 1)                        # (a wrong max_len)
    q = queries(gen, 201, 2 * 70, 64, FP16)
    run(PROMPT, q, k, v, scales, wide(table, 16), seq, cu, 200)                   # one token has more than 64 rows
    cache.attention(q[:0], k, v, scales, table, seq, ints([0, 0, 0]))
    assert capi.load().i4mm_last_attention_kernels() == 0


@pytest.mark.parametrize("held,dtype", [(INT8, FP16), (E4M3, BF16)])
@pytest.mark.parametrize("heads,group,dim", [(2, 8, 128), (4, 4, 64), (1, 70, 128)])
@pytest.mark.parametrize("window", [1, 5, 16, 100, 128, 129, 200, 257, 1000])
def test_windows_in_the_prompt_kernel(window, heads, group, dim, held, dtype):
    """Windows that end inside a tile, hide whole tiles from some rows of a tile of rows, and begin before the first token."""
    lens, seqs = [200, 1, 129, 150, 140], [200, 700, 1500, 151, 1024]
    k, v, scales, table, gen = make(seqs, heads, 16, dim, held, window + group)
    run(PROMPT if group > 64 else BOTH, queries(gen, sum(lens), heads * group, dim, dtype), k, v, scales, table if window < 1000 else wide(table, 16), ints(seqs),
        packed(lens), max(lens), window=window)


@pytest.mark.parametrize("window", [0, 7, 140])
def test_windows_over_absent_pages_and_short_requests(window):
    """Rows of the prompt kernel that see nothing: hidden pages, and rows before the request's first token."""
    lens, seqs = [160, 130, 200], [100, 900, 1300]
    k, v, scales, table, gen = make(seqs, 2, 16, 128, INT8, window)
    table[1, 40:56] = -1
    table[2, 70:] = 2 ** 30
    got = run(BOTH, queries(gen, sum(lens) + 5, 16, 128, FP16), k, v, scales, wide(table, 16), ints(seqs), packed(lens), max(lens), window=window)
    assert (got[:60] == 0).all() and (got[sum(lens):] == 0).all()


@pytest.mark.parametrize("scale", [-0.09, -1e-30, 0.0, -2.0])
@pytest.mark.parametrize("held,dtype", [(INT8, FP16), (INT8, BF16), (E4M3, FP16), (E4M3, BF16)])
@pytest.mark.parametrize("dim", [64, 128])
def test_scales_that_are_negative_or_zero(dim, held, dtype, scale):
    for lens, seqs in (([1, 1, 1], [300, 1, 77]), ([3, 1, 2], [300, 1, 77]), ([200, 1, 150], [900, 1, 150])):
        k, v, scales, table, gen = make(seqs, 2, 16, dim, held, dim)
        q = queries(gen, sum(lens), 8, dim, dtype)
        run(FEW, q, k, v, scales, table, ints(seqs), packed(lens), max(lens) if max(lens) < 17 else 1, scale)
        if max(lens) > 64:
            run(BOTH, q, k, v, scales, wide(table, 16), ints(seqs), packed(lens), max(lens), scale)


def test_a_cache_whose_offsets_pass_32_bits_in_the_prompt_kernel():
    """4.3 GB of keys: the last pages lie beyond 2^32 bytes."""
    heads, page, dim = 8, 128, 128
    pages = (2 ** 32) // (heads * page * dim) + 40
    k, v = (torch.zeros((pages, heads, page, dim), dtype=INT8, device="cuda") for _ in range(2))
    scales = torch.full((pages, heads, 2), 2.0 ** -6, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(2)
    x = queries(gen, 400, 2 * heads, dim, FP16)
    ids = [pages - 1, 3, pages - 30, pages - 2]
    cache.write(k, v, scales, x[:, :heads], x[:, heads:], ints([ids[p // page] * page + p % page for p in range(400)]))
    sub = torch.tensor(ids, device="cuda")
    q = queries(gen, 300, heads, dim, FP16)
    got = cache.attention(q, k, v, scales, wide(ints([ids]), page), ints([400]), ints([0, 300]), 300)
    assert capi.load().i4mm_last_attention_kernels() == BOTH
    assert torch.equal(got, run(BOTH, q, k[sub].clone(), v[sub].clone(), scales[sub].clone(), wide(ints([[0, 1, 2, 3]]), page), ints([400]), ints([0, 300]), 300))
