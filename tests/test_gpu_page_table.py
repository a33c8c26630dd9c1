"""GPU: PageTable over several steps: captured ones, ones that are short of pages, ones that are taken back."""
import pytest
import torch

from cache_reference import plan as reference
from int4matmul_kernels_b200 import cache

pytestmark = pytest.mark.gpu


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def test_a_captured_step_goes_on_by_itself():
    """Every replay is the next step: lengths, pages and slots as those of as many plain steps."""
    t = cache.PageTable(3, 40, 16, 160)
    t.step(ints([20, 0, 31]), 51)
    seq, table, stack = t.seq_lens.tolist(), t.block_table.tolist(), list(range(39, -1, -1))[:t.free_count.item()]
    new = ints([1, 1, 2])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        p = t.step(new, 4)
    for i in range(30):
        if i == 20:
            new.copy_(ints([-1, 1, 0]))
        graph.replay()
        want = reference(seq, new.tolist(), table, stack, 16, 10, 4)
        seq, table, stack = want["lens"], want["table"], want["pushed"][:want["free"]]
        assert p.slots.tolist() == want["slots"] and p.missing.item() == 0
        assert t.seq_lens.tolist() == seq and t.block_table.tolist() == table and t.free_count.item() == len(stack)
