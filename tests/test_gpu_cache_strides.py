"""GPU: strides of a single page, head or token, whatever they are."""
import pytest
import torch

from int4matmul_kernels_b200 import cache, ops

pytestmark = pytest.mark.gpu


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def odd(t, dim, stride):
    """The same values with another stride of a dimension of size 1."""
    s = list(t.stride())
    s[dim] = stride
    return t.as_strided(t.shape, s)


@pytest.mark.parametrize("compiled", [True, False])
@pytest.mark.parametrize("held", [torch.int8, torch.float8_e4m3fn])
def test_any_stride(held, compiled, monkeypatch):
    if not compiled:
        monkeypatch.setattr(ops, "_native", False)
    gen = torch.Generator(device="cuda").manual_seed(1)
    for pages, heads in ((1, 3), (5, 1), (1, 1)):
        n = 16 * pages - 3
        results = []
        for strange in (False, True):
            c = cache.PagedCache(pages, heads, 16, 64, held)
            k, v = c.k, c.v
            x = torch.randn((n + 1, 4 * heads, 64), device="cuda", generator=gen.manual_seed(2)).half()
            one = [x[n:, :2 * heads], x[n:, 2 * heads:3 * heads], x[n:, 3 * heads:]]
            if strange:
                for dim, size in ((0, pages), (1, heads)):
                    if size == 1:
                        k, v = odd(k, dim, 7), odd(v, dim, 1)
                one = [odd(t, 0, 3) for t in one]
                if heads == 1:
                    one[1:] = [odd(t, 1, 5) for t in one[1:]]
            slots = ints(range(n + 1))
            cache.write(k, v, c.scales, x[:n, 2 * heads:3 * heads], x[:n, 3 * heads:], slots[:n])
            cache.write(k, v, c.scales, one[1], one[2], slots[n:])
            table = ints([list(range(pages))])
            results.append([*cache.read(k, v, c.scales, slots), c.scales, cache.attention(one[0], k, v, c.scales, table, ints([n + 1])),
                            cache.attention(x[:, :2 * heads], k, v, c.scales, table, ints([n + 1]), ints([0, n + 1]), n + 1)])
        for a, b in zip(*results):
            assert torch.equal(a, b)
