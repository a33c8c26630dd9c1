"""GPU: the scratch of attention over shared prefixes may hold anything before the call."""
import ctypes
import math

import pytest
import torch

from cache_reference import attention_bound, values
from int4matmul_kernels_b200 import cache, capi
from shared_reference import attention as reference
from test_gpu_cache_attention import BF16, E4M3, FP16, INT8, ints, make, queries
from test_gpu_cache_shared import sums

pytestmark = pytest.mark.gpu

# What stands for (first block, number of parts, row of a tile) beside a negative total: 148 blocks, tiles of 64 rows.  None of these names parts.
NO_PARTS = {"all": 0x00FFFFFF, "block 148": 0x00000194, "two from block 147": 0x00000293, "row 64": 0x00400100, "255 parts": 0x0000FF00, "beyond 24 bits": 0x01000100,
            "every bit": 0xFFFFFFFF, "none": 0x00000000}


def call(q, k, v, scales, table, seq, cu, max_len, of, starts, rows, scratch):
    lib, (pages, heads, page, dim) = capi.load(), k.shape
    c = capi.Cache(k.data_ptr(), v.data_ptr(), scales.data_ptr(), pages, heads, page, dim, *k.stride()[:3], *v.stride()[:3],
                   capi.CACHE_INT8 if k.dtype == INT8 else capi.CACHE_E4M3)
    ws = torch.zeros(lib.i4mm_cache_attention_workspace_bytes(), dtype=torch.uint8, device="cuda")
    out = torch.empty_like(q)
    status = lib.i4mm_cache_attention_shared(ctypes.byref(c), out.data_ptr(), q.data_ptr(), capi.TYPE_FP16 if q.dtype == FP16 else capi.TYPE_BF16, q.shape[0], q.shape[1],
                                             q.stride(0), q.stride(1), table.data_ptr(), table.shape[1], table.shape[1], seq.data_ptr(), cu.data_ptr(), seq.shape[0],
                                             max_len, 1 / math.sqrt(dim), 0, of.data_ptr(), starts.data_ptr(), rows.data_ptr(), rows.shape[0], scratch.data_ptr(),
                                             scratch.numel() * 4, ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream)
    assert status == capi.OK and lib.i4mm_device_status(ws.data_ptr(), torch.cuda.current_stream().cuda_stream) == capi.OK
    return out


def scratch_of(q, bits):
    """The totals (x = bits, total = -1) of all rows and heads, and sums of NaN."""
    floats = capi.load().i4mm_cache_shared_scratch_bytes(*q.shape) // 4
    scratch = torch.full((floats,), math.nan, device="cuda")
    scratch.view(torch.int32)[0:2 * q.shape[0] * q.shape[1]:2] = torch.tensor(bits, dtype=torch.int64).to(torch.int32)
    scratch[1:2 * q.shape[0] * q.shape[1]:2] = -1.0
    return scratch


# requests' tokens and new ones, query heads of a key head, key heads; which kernel works on the rows' own tokens
SHAPES = {
    "few rows, whole segments": ([200, 10, 20, 30], [0, 1, 1, 2], 2, 40, capi.ATTENTION_FEW_ROWS),
    "few rows, cut segments": ([200, 9000, 20, 3000], [0, 1, 1, 2], 2, 1, capi.ATTENTION_FEW_ROWS),
    "many rows": ([200, 160, 20, 300], [0, 150, 1, 130], 1, 8, capi.ATTENTION_PROMPT),
    "many rows, cut segments": ([200, 9000, 20, 3000], [0, 150, 1, 70], 1, 1, capi.ATTENTION_PROMPT),
    "many rows of single tokens": ([200, 900, 20, 300], [0, 1, 1, 2], 71, 1, capi.ATTENTION_PROMPT),
}


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("held,dtype,dim", [(INT8, FP16, 128), (E4M3, BF16, 64)])
def test_rows_that_no_list_names(shape, held, dtype, dim):
    """Rows whose request names a prefix, in a call whose lists are empty: no prefix kernel writes their totals.  They are rows without a prefix, and what the
    scratch holds in that place is no address."""
    seqs, lens, group, heads, kernel = SHAPES[shape]
    k, v, scales, table, gen = make(seqs, heads, 16, dim, held, 5)
    wide = torch.full((table.shape[0], table.shape[1] + 200000 // 16), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    table = wide if kernel == capi.ATTENTION_PROMPT else table
    q, seq, cu = queries(gen, sum(lens), heads * group, dim, dtype), ints(seqs), ints(sums(lens))
    out, size, reach, tail = reference(q, values(k, scales[..., 0]), values(v, scales[..., 1]), table, seq, cu, [-1] * 4, 1 / math.sqrt(dim))
    limit = attention_bound(out, size, reach, tail, dtype)
    for bits in NO_PARTS.values():
        got = call(q, k, v, scales, table, seq, cu, max(lens), ints([-1, 0, 0, 0]), ints([0] * 5), ints([-1] * sum(lens)), scratch_of(q, bits))
        assert capi.load().i4mm_last_attention_kernels() & kernel
        assert ((got.double() - out).abs() <= limit).all()


@pytest.mark.parametrize("held,dtype,dim", [(INT8, FP16, 128), (E4M3, BF16, 64)])
@pytest.mark.parametrize("prefix", [200, 30000])
def test_listed_rows(prefix, held, dtype, dim):
    """Lists as share makes them: what the scratch held is of no account, whether a prefix is joined or left in parts."""
    seqs, lens, of = [prefix, 130, 1, 50, 6], [0, 101, 1, 4, 1], [-1, 0, 0, 0, 0]
    k, v, scales, table, gen = make(seqs, 1, 64, dim, held, 3)
    q, seq, cu = queries(gen, sum(lens), 2, dim, dtype), ints(seqs), ints(sums(lens))
    shared = cache.share(ints(of), seq, cu, q.shape[0])
    out, size, reach, tail = reference(q, values(k, scales[..., 0]), values(v, scales[..., 1]), table, seq, cu, of, 1 / math.sqrt(dim))
    limit = attention_bound(out, size, reach, tail, dtype)
    want = cache.attention(q, k, v, scales, table, seq, cu, max(lens), shared=shared)
    for bits in NO_PARTS.values():
        got = call(q, k, v, scales, table, seq, cu, max(lens), *shared[:3], scratch_of(q, bits))
        assert torch.equal(got, want) and ((got.double() - out).abs() <= limit).all()
