"""GPU: steps of the server that cannot be made, or have nothing to add."""
import pytest
import torch

from int4matmul_kernels_b200 import serving, sharding

pytestmark = pytest.mark.gpu


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def server(pages=40, max_seq=160):
    cfg = sharding.StackConfig(hidden=256, mlp=512, layers=2, bits=4, group_size=64)
    return serving.CachedStack(sharding.DecoderStack(cfg, 0, 1, "cuda"), 4, pages, 16, 5, max_seq)


def rows(n, seed):
    return torch.randn((n, 256), device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).half()


def state(s):
    return [x.clone() for c in s.caches for x in (c.k, c.v, c.scales)] + [s.table.seq_lens.clone(), s.table.free_count.clone()]


# (new tokens, short of pages): 7 pages of 16, places of up to 160 tokens
SHORT = [([30, 17, 0, 0, 0], False), ([1, 1, 60, 0, 0], True), ([1, 1, 20, 0, 0], False), ([-1, 0, 0, 90, 0], True), ([3, 0, 1, 10, 20], True),
         ([-1, 1, 0, 5, 0], False), ([0, 140, 0, 1, 1], True), ([0, -1, 1, 1, 40], False), ([1, 1, 1, 1, 200], True), ([1, 0, -1, -1, 1], False)]


def test_a_server_that_runs_out_of_pages():
    """The caller is told; the step changes neither the table nor a cache; and what follows is what a server gives that never tried it."""
    s, plain = server(pages=7), server(pages=7)
    for i, (new, short) in enumerate(SHORT):
        h = rows(sum(max(n, 0) for n in new), i)
        before = state(s)
        out = s.step(h, ints(new), max(new))
        assert (s.plan.missing.item() > 0) == short, i
        if short:
            assert all(torch.equal(a, b) for a, b in zip(state(s), before)), i
        else:
            assert torch.equal(out, plain.step(h, ints(new), max(new))), i
            assert all(torch.equal(a, b) for a, b in zip(state(s), state(plain))), i
            table, seq = s.table.block_table.tolist(), s.table.seq_lens.tolist()
            used = [p for row, n in zip(table, seq) for p in row[:-(-n // 16)]]
            assert sorted(used + s.table.free_pages[:s.table.free_count.item()].tolist()) == list(range(7)), i


def test_rows_that_are_refused_leave_the_table_as_it_was():
    s = server()
    s.step(rows(6, 1), ints([3, 3, 0, 0, 0]), 3)
    seq, count = s.table.seq_lens.tolist(), s.table.free_count.item()
    for h, error in ((rows(5, 2).float(), TypeError), (rows(5, 2)[:, :128], ValueError), (rows(5, 2)[None], ValueError), (rows(5, 2).cpu(), ValueError)):
        with pytest.raises(error):
            s.step(h, ints([1, 1, 3, 0, 0]), 3)
        assert s.table.seq_lens.tolist() == seq and s.table.free_count.item() == count
    with pytest.raises(ValueError):
        s.step(rows(5, 2), ints([1, 1, 3, 0, 0]), -1)
    assert s.table.seq_lens.tolist() == seq


def test_a_step_in_which_requests_only_end():
    s, plain = server(), server()
    for x in (s, plain):
        x.step(rows(40, 3), ints([30, 3, 7, 0, 0]), 30)
    out = s.step(rows(0, 4), ints([-1, 0, -1, 0, 0]), 0)
    assert out.shape == (0, 256) and s.table.seq_lens.tolist() == [0, 3, 0, 0, 0] and s.table.free_count.item() == 39
    h = rows(3, 5)
    got, want = s.step(h, ints([0, 1, 0, 2, 0]), 2), plain.step(h, ints([-1, 1, -1, 2, 0]), 2)
    assert torch.equal(got, want)
    assert s.stack.forward(rows(0, 4)).shape == (0, 256)
