"""Norm and rotation of queries and keys with the store into the paged cache, against 64 bits. GPU only (-m gpu).

Bounds: a norm is a chain of d / 32 + 8 roundings of a relative 2^-24, a rotation three more of its pair's size, together under 24 x
2^-24 (|a| + |b|); a cache element is rounded once more, 2^-11 (f16) or 2^-8 (bf16) of it at most, 2^-25 where f16 has no smaller step."""
import pytest

from tests import serving_reference as ref

pytestmark = pytest.mark.gpu
ROUND = {"f16": (2.0**-11, 2.0**-25), "bf16": (2.0**-8, 0.0)}


def check(ctx, tokens, hq, hk, d, rotary, style, norm, dtype, page=16, offset=0, pad=0, order="heads", in_place=False, seed=0):
    import torch

    import recipe_dev_b200 as rq

    kind = {"f16": torch.float16, "bf16": torch.bfloat16}[dtype]
    gen = torch.Generator(device="cuda").manual_seed(seed)
    width = (hq + 2 * hk) * d + pad
    qkv = torch.randn(tokens * width + offset, generator=gen, device="cuda")[offset:].view(tokens, width)
    q, k, v = qkv[:, : hq * d], qkv[:, hq * d : (hq + hk) * d], qkv[:, (hq + hk) * d : (hq + 2 * hk) * d]
    q0, k0, v0 = (a.double().reshape(tokens, -1, d) for a in (q, k, v))
    gains = (1.0 + 0.2 * torch.randn((2, d), generator=gen, device="cuda")) if norm else (None, None)
    rows = 100
    table = ctx.rope_table(rows, rotary) if rotary else None
    pages = ref.pages(tokens, page) + 2
    shape = (pages, hk, page, d) if order == "heads" else (pages, page, hk, d)
    kc, vc = (torch.full(shape, 7.0, dtype=kind, device="cuda") for _ in range(2))
    cache = rq.KvCache(kc, vc) if order == "heads" else rq.KvCache(kc.transpose(1, 2), vc.transpose(1, 2))
    positions = torch.randint(0, rows, (tokens,), generator=gen, device="cuda").int()
    slots = torch.randperm(pages * page, generator=gen, device="cuda")[:tokens].int()
    if tokens > 4:
        positions[1], positions[2] = -5, rows + 3  # clamped
        slots[3], slots[4] = -1, pages * page  # passed over
    out = ctx.rope_store(q, k, v, positions, slots, table, cache, *gains, style=style, q_out=q if in_place else None)
    ctx.check()
    angles = (table if rotary else torch.zeros((rows, 0), device="cuda"))[positions.long().clamp(0, rows - 1)]
    want, size = ref.turned(q0, gains[0], 1e-6, angles, style)
    assert ((out.double().reshape(tokens, hq, d) - want).abs() <= 24 * 2.0**-24 * size + 1e-30).all()
    keys, size = ref.turned(k0, gains[1], 1e-6, angles, style)
    rel, least = ROUND[dtype]
    stored_k, stored_v = (torch.full((pages, hk, page, d), 7.0, dtype=torch.float64, device="cuda") for _ in range(2))
    slack = torch.zeros_like(stored_k)
    good = (slots >= 0) & (slots < pages * page)
    block, line = slots[good].long() // page, slots[good].long() % page
    stored_k[block, :, line], stored_v[block, :, line], slack[block, :, line] = keys[good], v0[good], 24 * 2.0**-24 * size[good]
    for got, exact, more in ((cache.k, stored_k, slack), (cache.v, stored_v, 0.0)):
        assert ((got.double() - exact).abs() <= (rel * exact.abs()).clamp(min=least) + 1.01 * more).all()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("style", ["halves", "pairs"])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_head_sizes_styles_and_types(rq_ctx, d, style, norm, dtype):
    check(rq_ctx, 33, 6, 2, d, d, style, norm, dtype)


@pytest.mark.parametrize("d,rotary", [(64, 0), (64, 16), (64, 48), (128, 0), (128, 32), (128, 64), (128, 112), (256, 64), (256, 80), (256, 240)])
@pytest.mark.parametrize("style", ["halves", "pairs"])
def test_part_of_a_head_is_rotated(rq_ctx, d, rotary, style):
    check(rq_ctx, 7, 3, 1, d, rotary, style, True, "f16")


@pytest.mark.parametrize("tokens,hq,hk", [(1, 1, 1), (1, 32, 8), (2, 40, 2), (64, 32, 8), (1021, 5, 5), (300, 71, 1)])
@pytest.mark.parametrize("page", [1, 16, 4096])
def test_tokens_heads_and_pages(rq_ctx, tokens, hq, hk, page):
    check(rq_ctx, tokens, hq, hk, 128, 128, "halves", True, "bf16", page=page)


@pytest.mark.parametrize("offset,pad", [(0, 1), (1, 0), (2, 3), (3, 4), (4, 4)])
@pytest.mark.parametrize("d", [64, 256])
def test_alignment_strides_and_layouts(rq_ctx, offset, pad, d):
    check(rq_ctx, 19, 4, 2, d, d, "pairs", True, "f16", offset=offset, pad=pad, order="lines")


def test_queries_in_place(rq_ctx):
    check(rq_ctx, 50, 8, 2, 128, 128, "halves", True, "f16", in_place=True)


def test_a_table_of_long_contexts(rq_ctx):
    """The angle of position 131071 is rounded once: in 32 bits its product would be off by up to 2^-8."""
    import math

    table = rq_ctx.rope_table(131072, 128, base=500000.0, frequency_scale=0.25).double().cpu()
    for p in (0, 1, 4095, 131071):
        for i in (0, 1, 31, 63):
            a = p * 0.25 * 500000.0 ** (-i / 64)
            assert abs(table[p, i] - math.cos(a)) <= 2.0**-24 and abs(table[p, 64 + i] - math.sin(a)) <= 2.0**-24


def test_refusals(rq_ctx):
    import torch

    import recipe_dev_b200 as rq

    x = torch.zeros((4, 256), device="cuda")
    i = torch.zeros(4, dtype=torch.int32, device="cuda")
    cache = rq.KvCache.empty(2, 2, 16, 128)
    table = rq_ctx.rope_table(8, 128)
    with pytest.raises(rq.RqError, match="multiple of 16"):
        rq_ctx.rope_store(x, x, x, i, i, torch.zeros((8, 24), device="cuda"), cache)
    with pytest.raises(rq.RqError, match="up to head_dim"):
        rq_ctx.rope_store(x, x, x, i, i, torch.zeros((8, 144), device="cuda"), cache)
    with pytest.raises(rq.RqError, match="epsilon"):
        rq_ctx.rope_store(x, x, x, i, i, table, cache, epsilon=-1.0)
    with pytest.raises(ValueError):
        rq_ctx.rope_store(x[:, :200], x, x, i, i, table, cache)
    with pytest.raises(ValueError):
        rq_ctx.rope_store(x, x[:, :128], x, i, i, table, cache)
    with pytest.raises(ValueError):
        rq_ctx.rope_store(x, x, x, i[:3], i, table, cache)
    with pytest.raises(ValueError):
        rq.KvCache(torch.zeros((2, 2, 16, 128), device="cuda"), torch.zeros((2, 2, 16, 128), device="cuda"))
    with pytest.raises(rq.RqError, match="64, 128 or 256"):
        rq_ctx.rope_store(x[:, :96], x[:, :96], x[:, :96], i, i, None, rq.KvCache.empty(2, 1, 16, 96))
    with pytest.raises(rq.RqError, match="power of two"):
        rq_ctx.rope_store(x, x, x, i, i, table, rq.KvCache.empty(2, 2, 12, 128))
    with pytest.raises(rq.RqError, match="multiple of 16 up to 256"):
        rq_ctx.rope_table(8, 40)
    big = torch.empty(8 * 16 * 128 + 4, dtype=torch.float16, device="cuda")
    skewed = big[1:-3].view(4, 2, 16, 128)
    with pytest.raises(rq.RqError, match="16-byte aligned"):
        rq_ctx.rope_store(x, x, x, i, i, table, rq.KvCache(skewed, skewed))
    rq_ctx.check()
