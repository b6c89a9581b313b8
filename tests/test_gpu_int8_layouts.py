"""Caches of 8-bit codes whose scales lie in another order than the codes, apart from one another, at any 4-byte address. GPU only (-m gpu).

Bounds: test_gpu_int8_cache.py's."""
import pytest

from tests.test_gpu_int8_cache import batch, compare, run

pytestmark = pytest.mark.gpu

# (order of pages, heads and lines; every how many floats; floats before the first)
ORDERS = [((0, 1, 2), 1, 1), ((0, 2, 1), 1, 3), ((1, 0, 2), 2, 1), ((2, 1, 0), 1, 0), ((1, 2, 0), 3, 2)]


def apart(scales, order, every, offset):
    """The same scales in a plane of their own, with what lies between them."""
    import torch

    shape = [scales.shape[i] for i in order]
    plane = torch.full((offset + scales.numel() * every,), 77.0, device="cuda")
    mine = plane[offset:].view(*shape, every)[..., 0].permute([order.index(i) for i in range(3)])
    mine.copy_(scales)
    return plane, mine


@pytest.mark.parametrize("order,every,offset", ORDERS)
@pytest.mark.parametrize("fresh,d", [(1, 64), (1, 128), (2, 256), (6, 128), (30, 64), (70, 128)])
def test_attention(rq_ctx, order, every, offset, fresh, d):
    import recipe_dev_b200 as rq

    b = batch([100, 3], [fresh, fresh], 4, 2, d, 16, seed=fresh, order="lines")
    c = b["cache"]
    compare(run(rq_ctx, dict(b, cache=rq.KvCache(c.k, c.v, apart(c.k_scale, order, every, offset)[1], apart(c.v_scale, order, every, offset)[1]))), b)


@pytest.mark.parametrize("order,every,offset", ORDERS)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hq,hk", [(4, 2), (3, 5)])
def test_store(rq_ctx, order, every, offset, d, hq, hk):
    """The same codes and scales as into a cache in one order, and nothing between the scales."""
    import torch

    import recipe_dev_b200 as rq

    gen = torch.Generator(device="cuda").manual_seed(d)
    tokens, pages, page = 37, 4, 16
    q, k, v = (torch.randn((tokens, n * d), generator=gen, device="cuda") for n in (hq, hk, hk))
    table, gain = rq_ctx.rope_table(64, d), 1.0 + 0.2 * torch.randn(d, generator=gen, device="cuda")
    positions = torch.arange(tokens, dtype=torch.int32, device="cuda")
    slots = torch.randperm(pages * page, generator=gen, device="cuda")[:tokens].int()
    slots[3], slots[5] = -1, pages * page

    def codes():
        return [torch.full((pages, hk, page, d), 7, dtype=torch.int8, device="cuda") for _ in range(2)]

    scales = [torch.full((pages, hk, page), 0.5, device="cuda") for _ in range(2)]
    planes = [apart(s, order, every, offset) for s in scales]
    plain, far = rq.KvCache(*codes(), *scales), rq.KvCache(*codes(), *(mine for _, mine in planes))
    for cache in (plain, far):
        rq_ctx.rope_store(q, k, v, positions, slots, table, cache, gain, gain)
    rq_ctx.check()
    for name in ("k", "v", "k_scale", "v_scale"):
        assert torch.equal(getattr(plain, name), getattr(far, name))
    for plane, _ in planes:
        rest = torch.ones(plane.shape, dtype=torch.bool, device="cuda")
        rest[offset::every] = False
        assert (plane[rest] == 77.0).all()


def test_a_recorded_store_passes_over_slots_that_are_outside(rq_ctx):
    import torch

    import recipe_dev_b200 as rq

    gen = torch.Generator(device="cuda").manual_seed(3)
    tokens, pages, page, hk, d = 6, 3, 16, 2, 128
    cache = rq.KvCache(*(torch.full((pages, hk, page, d), 7, dtype=torch.int8, device="cuda") for _ in range(2)), *(torch.full((pages, hk, page), 0.5, device="cuda") for _ in range(2)))
    q, k, v = (torch.randn((tokens, n * d), generator=gen, device="cuda") for n in (4, hk, hk))
    q_out, at, slots = torch.empty_like(q), torch.arange(tokens, dtype=torch.int32, device="cuda"), torch.full((tokens,), -1, dtype=torch.int32, device="cuda")
    rq_ctx.rope_store(q, k, v, at, slots, None, cache, q_out=q_out)
    torch.cuda.synchronize()
    rq_ctx.rope_store(q, k, v, at, slots, None, cache, q_out=q_out, stream=rq_ctx.sequence_begin())
    sequence = rq_ctx.sequence_end()
    written = torch.zeros((pages, page), dtype=torch.bool, device="cuda")
    for given in ([-1] * 6, [5, -1, 47, 48, 2**31 - 1, 20], [-(2**31), 6, -1, 30, 31, 1000]):
        slots.copy_(torch.tensor(given, dtype=torch.int32))
        for a in (q, k, v):
            a.normal_(generator=gen)
        sequence.run()
        torch.cuda.synchronize()
        assert torch.equal(q_out, q)
        for t, slot in enumerate(given):
            if 0 <= slot < pages * page:
                written[slot // page, slot % page] = True
                for x, codes, scales in ((k, cache.k, cache.k_scale), (v, cache.v, cache.v_scale)):
                    of = x[t].view(hk, d)
                    step = (of.abs().amax(1).double() / 127).float()
                    assert torch.equal(scales[slot // page, :, slot % page], step)
                    assert ((codes[slot // page, :, slot % page].double() * step.double()[:, None] - of.double()).abs() <= (0.5 + 2.0**-16) * step.double()[:, None]).all()
        for codes, scales in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
            others = ~written[:, None].expand(scales.shape)
            assert (codes[others] == 7).all() and (scales[others] == 0.5).all()
    sequence.free()
    rq_ctx.check()
