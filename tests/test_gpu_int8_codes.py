"""Codes of the 8-bit store, bit for bit: x / scale rounded to the nearest whole number, ties to even. GPU only (-m gpu).

What is expected is the quotient in 64 bits, rounded: it is the same whole number. Where a quotient of fp32 numbers is not h / 2 for a whole number h, 2 x - h scale is at least
the smaller of the two terms' last places, 2^-24 of the scale and more (x is half a scale or more there), so that the quotient lies 2^-25 or more from h / 2: 64 bits are off by 127 x 2^-53 at
most."""
import pytest

pytestmark = pytest.mark.gpu


def codes_of(ctx, x, pairs=True):
    """x [tokens, d] as the keys and the values of one head: codes and scales, the same for both."""
    import torch

    import recipe_dev_b200 as rq

    tokens, d = x.shape
    cache = rq.KvCache(*(torch.zeros((-(-tokens // 16), 1, 16, d), dtype=torch.int8, device="cuda") for _ in range(2)), *(torch.zeros((-(-tokens // 16), 1, 16), device="cuda") for _ in range(2)))
    at = torch.arange(tokens, dtype=torch.int32, device="cuda")
    ctx.rope_store(x, x, x, at, at, None, cache)
    ctx.check()
    assert torch.equal(cache.k, cache.v) and torch.equal(cache.k_scale, cache.v_scale)
    return cache.k.reshape(-1, d)[:tokens], cache.k_scale.reshape(-1)[:tokens]


def compare(ctx, x):
    import torch

    codes, scales = codes_of(ctx, x)
    want = (x.abs().amax(1).double() / 127.0).float()
    want[want < 2.0**-126] = 0.0
    assert torch.equal(scales, want)
    exact = torch.where(scales[:, None] == 0, 0.0, torch.round(x.double() / torch.where(scales == 0, 1.0, scales.double())[:, None]))
    assert torch.equal(codes.double(), exact), int((codes.double() != exact).sum())


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("power", [0, -100, -119, 60, 119])
def test_next_to_borders_and_at_them(rq_ctx, d, power):
    """Numbers as near to half a code more than a whole one as fp32 has them, on both sides, and ties where the scale is a power of two or has few bits."""
    import torch

    gen = torch.Generator(device="cuda").manual_seed(d + power)
    rows = 4000
    largest = 127.0 * torch.exp2(torch.rand(rows, generator=gen, device="cuda"))
    largest[::4] = 127.0 * (1 + torch.randint(0, 256, largest[::4].shape, generator=gen, device="cuda") / 256)
    largest[::16] = 127.0
    scale = (largest.double() / 127.0).float().double()
    border = torch.randint(-127, 127, (rows, d), generator=gen, device="cuda").double() + 0.5
    x = (border * scale[:, None]).float()
    steps = torch.randint(-2, 3, (rows, d), generator=gen, device="cuda", dtype=torch.int32)
    x = (x.view(torch.int32) + steps).view(torch.float32)
    at = torch.randint(0, d, (rows,), generator=gen, device="cuda")
    x[torch.arange(rows, device="cuda"), at] = largest
    compare(rq_ctx, x * 2.0**power)


@pytest.mark.parametrize("tokens,d", [(1, 64), (3, 128), (40000, 128)])
def test_normal_numbers(rq_ctx, tokens, d):
    import torch

    compare(rq_ctx, torch.randn((tokens, d), generator=torch.Generator(device="cuda").manual_seed(tokens), device="cuda"))


def test_heads_of_zeros_and_next_to_nothing(rq_ctx):
    import torch

    x = torch.randn((40, 128), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    x[::3] = 0.0
    x[1::3] *= 2.0 ** torch.linspace(-124, -112, x[1::3].shape[0], device="cuda")[:, None]
    x[5, 1:] = -0.0
    compare(rq_ctx, x)
