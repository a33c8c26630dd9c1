"""GPU: attention called by several host threads on one stream, which share its scratch."""
import threading

import pytest
import torch

from int4matmul_kernels_b200 import cache, ops
from test_gpu_cache_attention import FP16, INT8, ints, make, queries
from test_gpu_cache_shared import sums

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("compiled", [True, False])
def test_calls_of_two_threads_on_one_stream(compiled, monkeypatch):
    """Calls with prefixes left in parts, with many readers, and without prefixes, in any order: each of them has its own results."""
    if not compiled:
        monkeypatch.setattr(ops, "_native", False)
    calls = []

    def add(seqs, lens, of, heads, group, seed):
        k, v, scales, table, gen = make(seqs, heads, 16, 128, INT8, seed)
        q, seq, cu = queries(gen, sum(lens), heads * group, 128, FP16), ints(seqs), ints(sums(lens))
        shared = cache.share(ints(of), seq, cu, sum(lens)) if of else None
        calls.append(lambda: cache.attention(q, k, v, scales, table, seq, cu, max(lens), shared=shared))

    add([20000, 900, 1500, 700], [0, 1, 1, 2], [-1, 0, 0, 0], 1, 4, 1)        # all blocks have a part of the prefix
    add([500] + [20 + i for i in range(40)], [0] + [1] * 40, [-1] + [0] * 40, 4, 8, 2)       # 320 rows of a key head
    add([3000, 40, 1200], [1, 1, 1], None, 4, 2, 3)
    add([700, 300], [1, 200], None, 2, 2, 4)
    want = [call() for call in calls]
    torch.cuda.synchronize()
    wrong, begin = [], threading.Barrier(2)

    def work(order):
        try:
            begin.wait(60)
            for _ in range(40):
                got = [(i, calls[i]()) for i in order]
                wrong.extend(i for i, x in got if not torch.equal(x, want[i]))
        except Exception as e:                                                # (a thread's failure is the test's)
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(order,)) for order in ([0, 1, 2, 3, 0, 2], [2, 0, 3, 2, 1, 0])]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong[:5]
    ops.check_device_status()
