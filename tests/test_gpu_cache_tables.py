"""GPU: angles of positions against 64 bits, and the tables of shared prefixes against plain Python."""
import math
import random

import pytest
import torch

from int4matmul_kernels_b200 import cache, ops
from shared_reference import share as reference

pytestmark = pytest.mark.gpu


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("tokens", [1, 2, 7, 64, 1000, 70001])
@pytest.mark.parametrize("pairs,theta", [(8, 100.0), (24, 10000.0), (64, 500000.0), (128, 10000.0)])
def test_angles(tokens, pairs, theta):
    """Errors: the argument's rounding to fp32, 2^-25 of half a turn; the fp32 functions, 2 units, 2^-23; and three fp64 roundings of the number
    of turns, 2^-51 of it."""
    gen = torch.Generator(device="cuda").manual_seed(tokens + pairs)
    positions = torch.randint(0, 2 ** 31 - 1, (tokens,), device="cuda", generator=gen, dtype=torch.int32)
    positions >>= torch.randint(0, 31, (tokens,), device="cuda", generator=gen, dtype=torch.int32)
    positions[:2] = ints([0, 2 ** 31 - 1])[:tokens]
    if tokens > 5:
        positions[5] = -1
    freqs = (theta ** (-torch.arange(pairs, dtype=torch.float64) / pairs)).float().cuda()
    got = cache.angles(positions, freqs)
    assert got.shape == (tokens, pairs, 2) and got.dtype == torch.float32
    a = positions.clamp(min=0).double()[:, None] * freqs.double()
    want = torch.stack([a.cos(), a.sin()], -1)
    limit = math.pi * 2.0 ** -25 + 2.0 ** -23 + 2.0 ** -51 * a[..., None]
    assert ((got.double() - want).abs() <= limit).all()
    assert (got[positions < 0] == torch.tensor([1.0, 0.0], device="cuda")).all()


def test_angles_of_any_frequency():
    """Above one turn a token, and backwards."""
    positions = torch.arange(300, dtype=torch.int32, device="cuda")
    freqs = torch.tensor([0.0, 7.25, -0.5, 1e3, 2.0 ** -140, 1.0, 6.2831855, -3.1415927], device="cuda")
    a = positions.double()[:, None] * freqs.double()
    got = cache.angles(positions, freqs).double()
    assert ((got - torch.stack([a.cos(), a.sin()], -1)).abs() <= math.pi * 2.0 ** -25 + 2.0 ** -23 + 2.0 ** -51 * a.abs()[..., None]).all()


def check(of, seq, cu, max_tokens):
    got = cache.share(ints(of), ints(seq), ints(cu), max_tokens)
    want = reference(of, seq, cu, max_tokens)
    for name, value in want.items():
        assert getattr(got, name).tolist() == value, name
    return got


def test_share_by_hand():
    # places 0 and 3 are prefixes; 1 and 4 read place 0, 5 reads 3; 2 has none; 6 names itself, 7 a place without tokens (8), 9 none of the batch
    got = check([-1, 0, -1, -1, 0, 3, 6, 8, -1, 10], [40, 5, 6, 20, 3, 9, 4, 4, 0, 2], [0, 0, 2, 3, 3, 4, 8, 9, 10, 10, 12], 16)
    assert got.rows.tolist()[:8] == [0, 1, 3, 4, 5, 6, 7, -1]
    assert got.positions.tolist()[:8] == [43, 44, 5, 42, 25, 26, 27, 28]


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 100, 511, 512, 513, 3000, 16384])
@pytest.mark.parametrize("most", [1, 70])
def test_share(n, most):
    rng = random.Random(n + most)
    new = [rng.choice([0, 1, 1, rng.randint(0, most)]) for _ in range(n)]
    seq = [rng.choice([0, c, c + rng.randint(0, 50), max(0, c - 3)]) for c in new]      # (some hold fewer tokens than they have rows)
    cu = [0]
    for c in new:
        cu.append(cu[-1] + c)
    few = [rng.randrange(n) for _ in range(5)]
    for of in ([rng.choice([-1, -7, n, rng.randrange(n)] + few) for _ in range(n)], [0] * n, list(range(n)), [n - 1 - b for b in range(n)]):
        check(of, seq, cu, cu[-1] + rng.choice([0, 5]))
    check(few[0:1] * n, seq, cu, cu[-1] // 2)                                           # rows beyond max_tokens have no entry


def test_nothing():
    got = cache.share(ints([]), ints([]), ints([0]), 3)
    assert got.prefix_of.numel() == 0 and got.starts.tolist() == [0] and got.rows.tolist() == [-1] * 3 and got.positions.tolist() == [-1] * 3
    assert cache.share(ints([-1]), ints([5]), ints([0, 0]), 0).rows.numel() == 0
    assert cache.angles(ints([]), torch.ones(8, device="cuda")).shape == (0, 8, 2)


def test_table_share_and_another_stream():
    table = cache.PageTable(4, 40, 16, 256)
    table.step(ints([50, 0, 0, 0]), 50)
    plan = table.step(ints([0, 3, 2, 1]), 8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        shared = table.share(ints([-1, 0, 0, -1]), plan)
        angles = cache.angles(shared.positions, torch.ones(8, device="cuda"))
    torch.cuda.current_stream().wait_stream(side)
    assert shared.rows.tolist() == [0, 1, 2, 3, 4, -1, -1, -1]
    assert shared.positions.tolist() == [50, 51, 52, 50, 51, 0, -1, -1]
    assert abs(float(angles[2, 3, 0]) - math.cos(52)) < 1e-6


def test_captured_tables_follow_their_inputs():
    of, seq, cu, freqs = ints([-1, 0, 0]), ints([30, 4, 9]), ints([0, 0, 2, 5]), torch.ones(8, device="cuda")
    cache.angles(cache.share(of, seq, cu, 8).positions, freqs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        shared = cache.share(of, seq, cu, 8)
        angles = cache.angles(shared.positions, freqs)
    of.copy_(ints([-1, -1, 0]))
    seq.copy_(ints([20, 2, 4]))
    graph.replay()
    torch.cuda.synchronize()
    want = reference([-1, -1, 0], [20, 2, 4], [0, 0, 2, 5], 8)
    assert {n: getattr(shared, n).tolist() for n in want} == want
    assert abs(float(angles[4, 0, 1]) - math.sin(23)) < 1e-6


def test_refusals():
    good = (ints([-1, 0]), ints([3, 4]), ints([0, 1, 2]), 4)
    cache.share(*good)
    for i, bad in ((0, ints([-1])), (1, ints([3])), (2, ints([0, 1])), (0, ints([[-1, 0]])), (3, -1)):
        with pytest.raises(ValueError):
            cache.share(*good[:i], bad, *good[i + 1:])
    with pytest.raises(TypeError):
        cache.share(good[0].long(), *good[1:])
    with pytest.raises(ValueError):
        cache.share(good[0].cpu(), *good[1:])
    with pytest.raises(ValueError):
        cache.share(ints([-1, 5, 0, 5])[::2], *good[1:])
    with pytest.raises(ops.Int4MatmulError):
        cache.share(ints([-1] * 16385), ints([1] * 16385), ints([0] * 16386), 4)
    freqs = torch.ones(16, device="cuda")
    for positions, f, error in ((ints([1]).long(), freqs, TypeError), (ints([[1]]), freqs, ValueError), (ints([1]), freqs.double(), TypeError),
                                (ints([1]), freqs.cpu(), ValueError), (ints([1]), freqs[::2], ValueError), (ints([1]), freqs[:4], ops.Int4MatmulError),
                                (ints([1]), torch.ones(136, device="cuda"), ops.Int4MatmulError), (ints([1]).cpu(), freqs, ValueError)):
        with pytest.raises(error):
            cache.angles(positions, f)
