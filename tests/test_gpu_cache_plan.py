"""GPU: the tables of a step against plain Python."""
import random

import pytest
import torch

from cache_reference import plan as reference
from int4matmul_kernels_b200 import cache, capi, ops

pytestmark = pytest.mark.gpu


def ints(v, shape=None):
    t = torch.tensor(v, dtype=torch.int32, device="cuda")
    return t.reshape(shape) if shape is not None else t


def problem(n, page, longest, most_new, ending, spare, seed, width=None):
    r = random.Random(seed)
    seq = [r.choice([0, 1, page - 1, page, page + 1, r.randint(0, longest)]) for _ in range(n)]
    new = [-1 if r.random() < ending else r.choice([0, 1, r.randint(0, most_new)]) for _ in range(n)]
    width = max([1] + [-(-(s + max(a, 0)) // page) for s, a in zip(seq, new)]) if width is None else width
    seq = [min(s, width * page) for s in seq]
    used = [-(-s // page) for s in seq]
    pages = sum(used) + spare
    order = r.sample(range(pages), pages)
    table, at = [], 0
    for u in used:
        table.append(order[at:at + u] + [-7] * (width - u))
        at += u
    return seq, new, table, order[at:], pages, width


def check(seq, new, table, stack, pages, width, page, max_tokens, capacity=None):
    want = reference(seq, new, table, stack, page, width, max_tokens)
    capacity = pages if capacity is None else capacity
    dev = dict(seq=ints(seq), new=ints(new), table=ints(table, (len(seq), width)), free=ints(stack + [-9] * (capacity - len(stack))),
               count=ints([len(stack)]))
    for _ in range(2):                                        # the same call again: the same answers
        p = cache.plan(dev["seq"], dev["new"], dev["table"], dev["free"], dev["count"], page, max_tokens)
        assert p.seq_lens.tolist() == want["lens"]
        assert p.cu_lens.tolist() == want["cu"]
        assert p.slots.tolist() == want["slots"]
        assert p.positions.tolist() == want["positions"]
        assert p.requests.tolist() == want["requests"]
        assert (p.free_count.item(), p.missing.item()) == (want["free"], want["missing"])
        assert dev["table"].tolist() == want["table"]
        assert dev["free"][:len(want["pushed"])].tolist() == want["pushed"]
        assert dev["seq"].tolist() == seq and dev["count"].item() == len(stack)
    return p, dev


@pytest.mark.parametrize("n,page,longest,most_new,ending,spare", [
    (1, 16, 0, 1, 0, 4), (1, 128, 5000, 1, 0, 1), (2, 16, 100, 700, 0, 99), (7, 32, 300, 1, 0.3, 9), (31, 64, 900, 40, 0.2, 60),
    (32, 16, 200, 0, 0.9, 5), (33, 16, 200, 5, 0, 200), (500, 64, 3000, 90, 0.1, 900), (513, 16, 90, 1, 0.1, 600), (1100, 16, 30, 9, 0.2, 2000),
    (5000, 16, 40, 2, 0.1, 6000)])
def test_tables_of_a_step(n, page, longest, most_new, ending, spare):
    for seed in range(3):
        case = problem(n, page, longest, most_new, ending, spare, seed + 10 * n)
        tokens = sum(max(a, 0) for a in case[1])
        for max_tokens in {tokens, tokens + 5, max(0, tokens - 3)}:
            check(*case, page, max_tokens)


def test_pages_that_run_out():
    for seed in range(4):
        case = problem(40, 16, 100, 60, 0.1, 11, seed)
        p, _ = check(*case, 16, 3000)
        assert p.missing.item() > 0 and p.free_count.item() == 0


def test_a_step_that_finds_no_pages_is_taken_back():
    t = cache.PageTable(3, 5, 16, 200)
    with pytest.raises(ValueError):
        t.undo()
    assert t.step(ints([30, 16, 0]), 46).missing.item() == 0
    assert t.step(ints([40, 1, 20]), 61).missing.item() == 4
    t.undo()
    assert t.seq_lens.tolist() == [30, 16, 0] and t.free_count.item() == 2
    p = t.step(ints([-1, 1, 40]), 41)
    assert p.missing.item() == 0 and p.free_count.item() == 0
    table = t.block_table.tolist()
    assert sorted(table[1][:2] + table[2][:3]) == [0, 1, 2, 3, 4] and p.slots.min().item() >= 0


def test_table_rows_that_are_full():
    for seed in range(4):
        check(*problem(9, 16, 100, 200, 0.1, 100, seed, width=4), 16, 2000)


def test_nothing_to_do_and_no_requests():
    check([0, 0, 0], [0, 0, 0], [[-1], [-1], [-1]], [4, 5], 6, 1, 16, 8)
    p = cache.plan(ints([]), ints([]), ints([], (0, 4)), ints([3, 1]), ints([2]), 16, 4)
    assert p.cu_lens.tolist() == [0] and p.slots.tolist() == [-1] * 4 and p.free_count.item() == 2 and p.missing.item() == 0


def test_pages_of_ended_requests_are_given_out_in_the_same_step():
    p, dev = check([40, 17, 0], [-1, 40, 70], [[5, 6, 7, -1, -1], [1, 2, -1, -1, -1], [-1] * 5], [9, 8], 10, 5, 16, 128)
    assert p.missing.item() == 2                          # 7 wanted, 5 there
    assert dev["table"][1].tolist()[:4] == [1, 2, 7, 6]


def test_a_row_of_a_wider_table():
    wide = torch.full((3, 12), -1, dtype=torch.int32, device="cuda")
    table = wide[:, 2:6]
    p = cache.plan(ints([0, 0, 0]), ints([20, 1, 0]), table, ints([0, 1, 2, 3]), ints([4]), 16, 24)
    assert table.tolist() == [[3, 2, -1, -1], [1, -1, -1, -1], [-1] * 4] and (wide[:, :2] == -1).all() and (wide[:, 6:] == -1).all()
    assert p.slots.tolist()[:21] == [48 + i for i in range(16)] + [32 + i for i in range(4)] + [16]


def test_other_streams_and_steps_in_a_row():
    """Steps that follow each other on a side stream, each taking the last one's Plan."""
    r = random.Random(3)
    n, page, width, pages = 20, 16, 30, 400
    seq, table, stack = [0] * n, [[-1] * width for _ in range(n)], list(range(pages))
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        dev = dict(seq=ints(seq), table=ints(table), free=ints(stack), count=ints([pages]))
        for step in range(8):
            new = [r.choice([-1, 0, 1, 1, 30]) for _ in range(n)]
            p = cache.plan(dev["seq"], ints(new), dev["table"], dev["free"], dev["count"], page, 700)
            dev["seq"], dev["count"] = p.seq_lens, p.free_count
            want = reference(seq, new, table, stack, page, width, 700)
            assert p.slots.tolist() == want["slots"], step
            assert dev["table"].tolist() == want["table"], step
            seq, table, stack = want["lens"], want["table"], want["pushed"][:want["free"]]


def test_refusals():
    a = (ints([1]), ints([1]), ints([[0, -1]]), ints([1]), ints([1]))
    cache.plan(*a, 16, 1)
    for i in range(5):
        with pytest.raises(ValueError):
            cache.plan(*a[:i], a[i].cpu(), *a[i + 1:], 16, 1)
        with pytest.raises(TypeError):
            cache.plan(*a[:i], a[i].long(), *a[i + 1:], 16, 1)
    with pytest.raises(ValueError):
        cache.plan(ints([1, 2]), *a[1:], 16, 1)
    with pytest.raises(ValueError):
        cache.plan(*a[:2], ints([0, 1]), *a[3:], 16, 1)
    with pytest.raises(ValueError):
        cache.plan(*a, 16, -1)
    for page in (0, 8, 24, 256, -16):
        with pytest.raises(ops.Int4MatmulError) as e:
            cache.plan(*a, page, 1)
        assert e.value.status == capi.ERR_UNSUPPORTED
    n = 16385
    with pytest.raises(ops.Int4MatmulError) as e:
        cache.plan(ints([0] * n), ints([0] * n), ints([[0]] * n), a[3], a[4], 16, 1)
    assert e.value.status == capi.ERR_SHAPE
