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


def filled(requests, pages, lens, max_seq=200):
    """A table whose requests have these lengths, a cache that holds their tokens, and their slots."""
    t, c = cache.PageTable(requests, pages, 16, max_seq), cache.PagedCache(pages, 2, 16, 64)
    p = t.step(ints(lens), sum(lens))
    gen = torch.Generator(device="cuda").manual_seed(7)
    x = torch.randn((sum(lens), 4, 64), device="cuda", generator=gen).half()
    c.write(x[:, :2], x[:, 2:], p.slots)
    return t, c, p.slots.clone()


def contents(c):
    return c.k.clone(), c.v.clone(), c.scales.clone()


@pytest.mark.parametrize("lens,short,fits", [([16, 16], [-1, 40], [-1, 8]), ([20, 11], [-1, 60], [2, 1]), ([20, 5], [12, 30], [0, -1]), ([10, 10], [200, 1], [1, 1])])
def test_a_step_short_of_pages_changes_nothing(lens, short, fits):
    """Its tokens are written and attended to as a program does that has not looked at Plan.missing; the pages of a request that would have ended, and
    places and scales of pages that were only added to, are what they were, with undo and without."""
    for undo in (False, True):
        pages = sum(-(-n // 16) for n in lens)
        t, c, slots = filled(2, pages, lens)
        before, held, seq = contents(c), c.read(slots), t.seq_lens.tolist()
        p = t.step(ints(short), sum(max(n, 0) for n in short))
        assert p.missing.item() > 0 and p.slots.max().item() == -1
        x = 100 * torch.ones((p.slots.shape[0], 4, 64), dtype=torch.float16, device="cuda")
        c.write(x[:, :2], x[:, 2:], p.slots)
        c.attention(x, t, p.cu_lens, max(short))
        if undo:
            t.undo()
        assert t.seq_lens.tolist() == seq and t.free_count.item() == 0
        for a, b in zip(contents(c), before):
            assert torch.equal(a, b)
        for a, b in zip(c.read(slots), held):
            assert torch.equal(a, b)
        # the same requests go on, and all pages are given out once
        p = t.step(ints(fits), sum(max(n, 0) for n in fits))
        assert p.missing.item() == 0 and (p.slots >= 0).all()
        table, now = t.block_table.tolist(), t.seq_lens.tolist()
        used = [i for row, n in zip(table, now) for i in row[:-(-n // 16)]]
        assert len(set(used)) == len(used) and sorted(used + t.free_pages[:t.free_count.item()].tolist()) == list(range(pages))


def test_undo_before_a_step_is_written():
    t, c, slots = filled(3, 8, [30, 17, 0])
    held, seq, count = c.read(slots), t.seq_lens.tolist(), t.free_count.item()
    assert t.step(ints([-1, 20, 40]), 60).missing.item() == 0
    t.undo()
    assert t.seq_lens.tolist() == seq and t.free_count.item() == count
    for a, b in zip(c.read(slots), held):
        assert torch.equal(a, b)
    with pytest.raises(ValueError):
        t.undo()
    # and the lengths' own storage stays: what was captured or kept goes on reading the table's
    kept = t.seq_lens
    t.step(ints([1, 0, 0]), 1)
    assert kept.tolist() == [31, 17, 0]


def test_tables_made_and_used_in_and_out_of_inference_mode():
    with torch.inference_mode():
        t = cache.PageTable(2, 8, 16, 64)
        t.step(ints([3, 0]), 3)
    t.step(ints([1, 20]), 21)
    with torch.inference_mode():
        assert t.step(ints([1, 1]), 2).slots.tolist() == [t.block_table[0, 0].item() * 16 + 4, t.block_table[1, 1].item() * 16 + 4]
        t.undo()
    assert t.seq_lens.tolist() == [4, 20] and t.free_count.item() == 5


def test_a_captured_step_that_runs_out_of_pages_stops():
    t = cache.PageTable(2, 5, 16, 160)
    t.step(ints([16, 30]), 46)
    new = ints([4, 4])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        p = t.step(new, 8)
    for want in ([20, 34], [24, 38], [28, 42], [32, 46], [32, 46], [32, 46]):        # (the next would be 36 and 50: 3 and 4 pages of 5)
        graph.replay()
        assert t.seq_lens.tolist() == want
        assert (p.missing.item() > 0) == (p.slots.max().item() < 0)
    assert p.missing.item() == 2 and t.free_count.item() == 0
    new.copy_(ints([-1, 4]))
    graph.replay()
    assert t.seq_lens.tolist() == [0, 50] and p.missing.item() == 0 and t.free_count.item() == 1
