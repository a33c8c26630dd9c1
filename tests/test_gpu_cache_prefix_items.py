"""GPU: attention over shared prefixes where a block works on many short segments, one right after the other."""
import pytest
import torch

from int4matmul_kernels_b200 import cache
from test_gpu_cache_attention import BF16, E4M3, FP16, INT8, ints, make, queries
from test_gpu_cache_shared import check, sums

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("held,dtype,dim,window", [(INT8, FP16, 128, 0), (E4M3, BF16, 128, 0), (INT8, FP16, 64, 0), (INT8, BF16, 128, 90)])
@pytest.mark.parametrize("prefix", [1, 128, 200, 256])
def test_segments_of_one_and_two_tiles(prefix, held, dtype, dim, window):
    """Twelve places under 32 heads are 384 segments: two or three for each block, of one tile or two, so that the queries of the next are looked for while
    those of this one are being loaded.  33 to 64 rows a segment, each request's queries far from its neighbours' (columns of a wide projection)."""
    places, heads = 12, 32
    readers = [33 + (7 * i) % 32 for i in range(places)]
    of = [-1] * places + [p for p, n in enumerate(readers) for _ in range(n)]
    own = [1 + i % 5 for i in range(sum(readers))]
    seqs, lens = [max(1, prefix - p % 3) for p in range(places)] + own, [0] * places + [1] * len(own)
    k, v, scales, table, gen = make(seqs, heads, 16, dim, held, prefix + dim)
    q = queries(gen, len(own), 3 * heads, dim, dtype)[:, heads:2 * heads]
    want = check(q, k, v, scales, table, seqs, lens, of, window=window)
    seq, cu = ints(seqs), ints(sums(lens))
    shared = cache.share(ints(of), seq, cu, len(own))
    cold = torch.empty(1 << 28, dtype=torch.int8, device="cuda")
    for i in range(40):
        if i % 4 == 0:
            cold.zero_()                                                      # the queries come from memory, some warps' long after the others'
        assert torch.equal(cache.attention(q, k, v, scales, table, seq, cu, 1, window=window, shared=shared), want)
