"""GPU: positions, head norms and shared prefixes where only the C ABI library is built (no compiled module)."""
import pytest
import torch

from int4matmul_kernels_b200 import cache, capi, ops

pytestmark = pytest.mark.gpu
FP16, BF16 = torch.float16, torch.bfloat16


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def steps(dtype, held, interleaved):
    """A system prompt, two requests behind it and one without, over three steps: every result on the way."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    table, c = cache.PageTable(4, 30, 16, 128), cache.PagedCache(30, 2, 16, 64, held)
    freqs = (1e4 ** (-torch.arange(24, dtype=torch.float64) / 24)).float().cuda()
    weight, results = torch.linspace(0.5, 1.5, 64, device="cuda").to(dtype), []
    for new in ([50, 0, 0, 0], [0, 20, 1, 3], [0, 1, 1, 1]):
        p = table.step(ints(new), sum(new) + 2)
        shared = table.share(ints([-1, 0, 0, -1]), p)
        angles = cache.angles(shared.positions, freqs)
        x = torch.randn((sum(new), 8, 64), device="cuda", generator=gen).to(dtype)
        q = c.append(x[:, :4], x[:, 4:6], x[:, 6:], p.slots, angles, q_weight=weight, k_weight=weight, eps=1e-5, interleaved=interleaved)
        results += [*shared, angles, q, c.attention(q, table, p.cu_lens, max(new), shared=shared, window=40), c.scales.clone(), c.k.view(torch.int8).clone()]
    q = c.append(x[:, :4], x[:, 4:6], x[:, 6:], ints([-1] * 3), k_weight=weight)                   # no rotation; nothing is written
    return results + [q, c.scales.clone()]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("held", [torch.int8, torch.float8_e4m3fn])
def test_both_ways_give_the_same(dtype, held, interleaved, monkeypatch):
    compiled = steps(dtype, held, interleaved)
    monkeypatch.setattr(ops, "_native", False)
    for a, b in zip(compiled, steps(dtype, held, interleaved), strict=True):
        assert torch.equal(a, b)


def test_no_gradients():
    c = cache.PagedCache(2, 2, 16, 64)
    q, kv = torch.randn((3, 2, 64), device="cuda").half().requires_grad_(), torch.randn((3, 2, 64), device="cuda").half()
    assert not c.append(q, kv, kv, ints([0, 1, 2]), cache.angles(ints([0, 1, 2]), torch.ones(8, device="cuda", requires_grad=True))).requires_grad


@pytest.mark.parametrize("native", [True, False])
def test_refusals(native, monkeypatch):
    if not native:
        monkeypatch.setattr(ops, "_native", False)
    c, x = cache.PagedCache(4, 2, 16, 64), torch.zeros((3, 2, 64), dtype=FP16, device="cuda")
    slots, angles = ints([0, 1, 2]), torch.zeros((3, 8, 2), device="cuda")
    for error, call in (
            (TypeError, lambda: c.append(x.float(), x, x, slots, angles)), (ValueError, lambda: c.append(x[:2], x, x, slots, angles)),
            (ValueError, lambda: c.append(x, x, x, slots[:2], angles)), (ValueError, lambda: c.append(x, x, x, slots, angles[:2])),
            (TypeError, lambda: c.append(x, x, x, slots, angles.half())), (ValueError, lambda: c.append(x, x, x, slots, angles, q_weight=x[0, 0, :32])),
            (ValueError, lambda: c.append(x, x, x, slots)), (TypeError, lambda: cache.angles(slots.long(), torch.ones(8, device="cuda"))),
            (TypeError, lambda: cache.angles(slots, torch.ones(8, device="cuda").half())), (ValueError, lambda: cache.angles(slots, torch.ones(8))),
            (ValueError, lambda: cache.share(slots, slots, slots, 3)), (ValueError, lambda: cache.share(slots, slots, ints([0, 1, 2, 3]), -1))):
        with pytest.raises(error):
            call()
    for call in (lambda: c.append(x, x, x, slots, torch.zeros((3, 12, 2), device="cuda")), lambda: cache.angles(slots, torch.ones(12, device="cuda"))):
        with pytest.raises(ops.Int4MatmulError) as e:
            call()
        assert e.value.status == capi.ERR_UNSUPPORTED
    assert (c.scales == 0).all()
