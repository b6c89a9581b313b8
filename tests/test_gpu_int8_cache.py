"""The cache of 8-bit codes with a scale for each position's head: the store into it, and attention over it, against 64 bits. GPU only (-m gpu).

Store: what is rounded lies within 24 x 2^-24 of its pair's size (test_gpu_rope_store.py); the scale is the largest magnitude over 127, another rounding; a code is off by half a step
and by three roundings of x / scale. Attention: the bound of each output is derived beside the reference (serving_reference.attention); scores and weights meet
one rounding more, the scale's, which the bound's 2 d (for d products) and 2^-18 (for weights of 22 bits) hold."""
import random

import pytest

from tests import serving_reference as ref

pytestmark = pytest.mark.gpu


def values(cache, name):
    import torch

    scale = getattr(cache, name + "_scale")
    return torch.where(scale[..., None] == 0, 0.0, getattr(cache, name).double() * scale.double()[..., None])


# ---- the store ---------------------------------------------------------------------------------------------


def store(ctx, tokens, hq, hk, d, rotary, style, norm, page=16, offset=0, pad=0, order="heads", seed=0, size=1.0):
    import torch

    import recipe_dev_b200 as rq

    gen = torch.Generator(device="cuda").manual_seed(seed)
    width = (hq + 2 * hk) * d + pad
    qkv = size * torch.randn(tokens * width + offset, generator=gen, device="cuda")[offset:].view(tokens, width)
    q, k, v = qkv[:, : hq * d], qkv[:, hq * d : (hq + hk) * d], qkv[:, (hq + hk) * d : (hq + 2 * hk) * d]
    if tokens > 6:
        k[5, :d], v[6, -d:] = 0.0, 0.0  # heads of zeros
    gains = (1.0 + 0.2 * torch.randn((2, d), generator=gen, device="cuda")) if norm else (None, None)
    rows = 100
    table = ctx.rope_table(rows, rotary) if rotary else None
    pages = ref.pages(tokens, page) + 2
    shape = (pages, hk, page) if order == "heads" else (pages, page, hk)
    planes = [torch.full((*shape, d), 7, dtype=torch.int8, device="cuda") for _ in range(2)] + [torch.full(shape, 0.5, device="cuda") for _ in range(2)]
    cache = rq.KvCache(*(a if order == "heads" else a.transpose(1, 2) for a in planes))
    positions = torch.randint(0, rows, (tokens,), generator=gen, device="cuda").int()
    slots = torch.randperm(pages * page, generator=gen, device="cuda")[:tokens].int()
    if tokens > 4:
        slots[3], slots[4] = -1, pages * page  # passed over
    out = ctx.rope_store(q, k, v, positions, slots, table, cache, *gains, style=style)
    ctx.check()
    angles = (table if rotary else torch.zeros((rows, 0), device="cuda"))[positions.long()]
    want, spread = ref.turned(q.double().reshape(tokens, -1, d), gains[0], 1e-6, angles, style)
    assert ((out.double().reshape(tokens, hq, d) - want).abs() <= 24 * 2.0**-24 * spread + 1e-30).all()
    keys, spread = ref.turned(k.double().reshape(tokens, -1, d), gains[1], 1e-6, angles, style)
    good = (slots >= 0) & (slots < pages * page)
    block, line = slots[good].long() // page, slots[good].long() % page
    touched = torch.zeros((pages, page), dtype=torch.bool, device="cuda")
    touched[block, line] = True
    for name, x, off in (("k", keys[good], 24 * 2.0**-24 * spread[good]), ("v", v.double().reshape(tokens, -1, d)[good], torch.zeros((), device="cuda"))):
        code, scale = getattr(cache, name), getattr(cache, name + "_scale")
        others = ~touched[:, None].expand(scale.shape)
        assert (code[others] == 7).all() and (scale[others] == 0.5).all()
        got, step = code[block, :, line].double(), scale[block, :, line].double()
        largest = x.abs().amax(-1)
        assert ((127 * step - largest).abs() <= off.expand(x.shape).amax(-1) * 1.01 + 2 * 2.0**-24 * largest).all()
        assert ((got * step[..., None] - x).abs() <= 0.5 * step[..., None] + 1.01 * off + 4 * 2.0**-24 * x.abs()).all()
        assert (got.abs().amax(-1) == torch.where(step > 0, 127, 0)).all() and (step[largest == 0] == 0).all()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("style", ["halves", "pairs"])
@pytest.mark.parametrize("norm", [False, True])
def test_store_head_sizes_and_styles(rq_ctx, d, style, norm):
    store(rq_ctx, 33, 6, 2, d, d, style, norm)


@pytest.mark.parametrize("d,rotary", [(64, 0), (64, 48), (128, 64), (256, 80)])
def test_store_part_of_a_head_is_rotated(rq_ctx, d, rotary):
    store(rq_ctx, 9, 3, 1, d, rotary, "halves", True)


@pytest.mark.parametrize("tokens,hq,hk", [(1, 1, 1), (1, 32, 8), (2, 40, 2), (3, 5, 5), (1021, 7, 3), (300, 71, 1)])
@pytest.mark.parametrize("page", [1, 16, 4096])
def test_store_tokens_heads_and_pages(rq_ctx, tokens, hq, hk, page):
    store(rq_ctx, tokens, hq, hk, 128, 128, "halves", True, page=page)


@pytest.mark.parametrize("offset,pad", [(0, 1), (1, 0), (2, 3), (4, 4)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_store_alignment_strides_and_layouts(rq_ctx, offset, pad, d):
    store(rq_ctx, 19, 4, 2, d, d, "pairs", True, offset=offset, pad=pad, order="lines")


@pytest.mark.parametrize("size", [2.0**-60, 2.0**-110, 2.0**60, 2.0**120])
def test_store_of_any_size(rq_ctx, size):
    store(rq_ctx, 20, 2, 2, 128, 0, "halves", False, size=size)


def test_store_of_heads_that_are_no_numbers_or_next_to_nothing(rq_ctx):
    import torch

    import recipe_dev_b200 as rq

    cache = rq.KvCache.empty(1, 1, 16, 64, torch.int8)
    x = torch.zeros((4, 64), device="cuda")
    x[0, 3], x[1, 5], x[2, 7], x[3, 9] = float("inf"), float("nan"), 1e-38, -1.0
    at = torch.arange(4, dtype=torch.int32, device="cuda")
    rq_ctx.rope_store(x, x, x, at, at, None, cache)
    scale = cache.k_scale[0, 0, :4].tolist()
    assert scale[0] == float("inf") and scale[1] != scale[1] and scale[2] == 0 and abs(scale[3] - 1 / 127) <= 2.0**-24 / 127
    assert cache.k[0, 0, 2].eq(0).all() and cache.k[0, 0, 3, 9] == -127 and cache.k[0, 0, 3].abs().sum() == 127


def test_a_prompt_leaves_the_same_bytes_as_its_tokens_one_by_one(rq_ctx):
    import torch

    import recipe_dev_b200 as rq

    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn((40, 3 * 256), generator=gen, device="cuda")
    table, gain = rq_ctx.rope_table(64, 128), 1.0 + 0.2 * torch.randn(128, generator=gen, device="cuda")
    at = torch.arange(40, dtype=torch.int32, device="cuda")
    caches = [rq.KvCache(*(torch.zeros(s, dtype=t, device="cuda") for t, s in ((torch.int8, (3, 2, 16, 128)),) * 2 + ((torch.float32, (3, 2, 16)),) * 2)) for _ in range(2)]
    q, k, v = x.split(256, dim=1)
    rq_ctx.rope_store(q, k, v, at, at, table, caches[0], gain, gain)
    for t in range(40):
        rq_ctx.rope_store(q[t : t + 1], k[t : t + 1], v[t : t + 1], at[t : t + 1], at[t : t + 1], table, caches[1], gain, gain)
    for name in ("k", "v", "k_scale", "v_scale"):
        assert torch.equal(getattr(caches[0], name), getattr(caches[1], name))


# ---- attention ---------------------------------------------------------------------------------------------


def batch(cached, fresh, hq, hk, d, page, seed=0, spread=2.0, order="heads", width=0, offset=0, pad=0, sizes=0.3):
    """A batch over randomly placed pages; every position past a request's length, and every page that nobody owns, holds codes of -128 and a scale of NaN."""
    import torch

    import recipe_dev_b200 as rq

    gen = torch.Generator(device="cuda").manual_seed(seed)
    lengths = [c + f for c, f in zip(cached, fresh)]
    held = [ref.pages(n, page) for n in lengths]
    total = sum(held) + 2
    shape = (total, hk, page) if order == "heads" else (total, page, hk)
    planes = [torch.full((*shape, d), -128, dtype=torch.int8, device="cuda") for _ in range(2)] + [torch.full(shape, float("nan"), device="cuda") for _ in range(2)]
    cache = rq.KvCache(*(a if order == "heads" else a.transpose(1, 2) for a in planes))
    ids = random.Random(seed).sample(range(total), sum(held))
    width = width or max(max(held), 1) + 1
    table = torch.full((len(cached), width + 3), 2**30, dtype=torch.int32, device="cuda")[:, :width]
    for r, n in enumerate(lengths):
        mine = [ids.pop() for _ in range(held[r])]
        for i, page_id in enumerate(mine[:width]):
            table[r, i] = page_id
        for i, page_id in enumerate(mine):
            lines = min(page, n - i * page)
            for codes, scales in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
                codes[page_id, :, :lines] = (42 * torch.randn((hk, lines, d), generator=gen, device="cuda")).round().clamp(-127, 127).to(torch.int8)
                scales[page_id, :, :lines] = torch.exp(sizes * torch.randn((hk, lines), generator=gen, device="cuda")) / 42
    tokens = sum(fresh)
    starts = [sum(fresh[:i]) for i in range(len(fresh) + 1)]
    q = torch.randn(tokens * (hq * d + pad) + offset, generator=gen, device="cuda")[offset:].view(tokens, hq * d + pad)[:, : hq * d]
    q.mul_(torch.linspace(0.3, spread, hq, device="cuda").repeat_interleave(d))
    return dict(q=q, cache=cache, table=table, starts=starts, lengths=lengths, hq=hq, d=d)


def run(ctx, b, window=0, scale=None, max_fresh=None, y=None):
    import torch

    def dev(a):
        return torch.tensor(a, dtype=torch.int32, device="cuda")

    fresh = max(e - s for s, e in zip(b["starts"], b["starts"][1:]))
    y = torch.full(b["q"].shape, 9.0, device="cuda") if y is None else y
    got = ctx.attention(b["q"], b["cache"], b["table"], dev(b["starts"]), dev(b["lengths"]), scale=scale, window=window, max_fresh=fresh if max_fresh is None else max_fresh, y=y)
    ctx.check()
    return got.reshape(-1, b["hq"], b["d"])


def compare(got, b, window=0, scale=None, norm=5e-6):
    import torch

    want, bound = ref.attention(b["q"].reshape(-1, b["hq"], b["d"]), values(b["cache"], "k"), values(b["cache"], "v"), b["table"], b["starts"], b["lengths"], scale or b["d"] ** -0.5, window)
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all() and (off <= bound).all(), float((off - bound).max())
    assert norm is None or off.norm() <= norm * want.norm()


@pytest.mark.parametrize("hq,hk,d", [(1, 1, 64), (8, 2, 128), (32, 8, 128), (4, 4, 256), (7, 1, 64), (20, 1, 128), (28, 4, 128), (40, 2, 64), (16, 1, 256), (128, 1, 64)])
def test_one_token_each(rq_ctx, hq, hk, d):
    b = batch([0, 1, 30, 299, 64, 127], [1] * 6, hq, hk, d, 16)
    compare(run(rq_ctx, b), b)


@pytest.mark.parametrize("hq,hk,d", [(8, 2, 128), (2, 2, 64), (6, 2, 256), (9, 3, 64), (24, 1, 128)])
def test_chunks_over_a_cache(rq_ctx, hq, hk, d):
    b = batch([0, 5, 130, 40, 0], [33, 1, 70, 0, 129], hq, hk, d, 16)
    compare(run(rq_ctx, b), b)


@pytest.mark.parametrize("page", [1, 2, 4, 8, 32, 64, 128, 256, 4096])
@pytest.mark.parametrize("fresh", [1, 3, 65])
def test_page_sizes(rq_ctx, page, fresh):
    b = batch([200, 0, 77], [fresh] * 3, 8, 2, 128, page)
    compare(run(rq_ctx, b), b)


@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 191, 193, 255, 256, 257, 383, 385])
def test_lengths_about_tile_ends(rq_ctx, length):
    for fresh in {1, min(length, 2), length}:
        b = batch([length - fresh], [fresh], 4, 2, 64, 16, seed=length)
        compare(run(rq_ctx, b), b)


@pytest.mark.parametrize("window", [1, 2, 17, 64, 100, 128, 1000])
def test_windows(rq_ctx, window):
    b = batch([0, 300, 63, 500], [40, 1, 130, 5], 4, 2, 128, 16)
    compare(run(rq_ctx, b, window=window), b, window=window)


@pytest.mark.parametrize("order,offset,pad", [("lines", 0, 0), ("heads", 1, 0), ("lines", 2, 5), ("heads", 4, 4)])
@pytest.mark.parametrize("fresh", [1, 40])
@pytest.mark.parametrize("d", [64, 128])
def test_layouts_alignment_and_strides(rq_ctx, order, offset, pad, fresh, d):
    import torch

    b = batch([60, 3], [fresh, fresh], 6, 2, d, 16, order=order, offset=offset, pad=pad)
    tokens = b["q"].shape[0]
    plane = torch.full((tokens * (6 * d + 7) + 1,), 5.0, device="cuda")
    y = plane[1:].view(tokens, 6 * d + 7)[:, : 6 * d]
    compare(run(rq_ctx, b, y=y), b)
    assert (plane[1:].view(tokens, -1)[:, 6 * d :] == 5.0).all() and plane[0] == 5.0


@pytest.mark.parametrize("fresh", [1, 9, 150])
def test_rows_that_see_nothing_and_pages_that_are_lacking(rq_ctx, fresh):
    b = batch([70, 0, 33], [fresh] * 3, 4, 2, 128, 16)
    b["table"][0, 1], b["table"][2, 0] = -1, 2**30  # pages outside the cache
    b["lengths"][1] = 0  # no positions at all: its tokens see nothing
    got = run(rq_ctx, b)
    assert (got[fresh : 2 * fresh] == 0).all()
    compare(got, b)


@pytest.mark.parametrize("fresh", [1, 4, 70])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_scales_that_differ_by_powers_of_two(rq_ctx, fresh, d):
    """A value of a small scale may weigh the most, and one of a large scale next to nothing, in one tile: no weight may lose its bits to another's scale."""
    import torch

    b = batch([150, 40], [fresh, fresh], 4, 2, d, 16, seed=fresh)
    gen = torch.Generator(device="cuda").manual_seed(1)
    c = b["cache"]
    c.v_scale.mul_(2.0 ** torch.randint(-40, 41, c.v_scale.shape, generator=gen, device="cuda"))
    compare(run(rq_ctx, b), b, norm=None)
    c.v_scale.mul_(2.0**-60)
    compare(run(rq_ctx, b), b, norm=None)
    c.v_scale.mul_(2.0**100)
    compare(run(rq_ctx, b), b, norm=None)


@pytest.mark.parametrize("fresh", [1, 70])
def test_keys_and_queries_of_any_size(rq_ctx, fresh):
    b = batch([100], [fresh], 4, 2, 128, 16)
    for q_size, k_size in ((2.0**-60, 2.0**60), (2.0**60, 2.0**-60), (2.0**-30, 2.0**30)):
        b["q"].mul_(q_size)
        b["cache"].k_scale.mul_(k_size)
        compare(run(rq_ctx, b), b)
        b["q"].mul_(1 / q_size)
        b["cache"].k_scale.mul_(1 / k_size)


@pytest.mark.parametrize("fresh", [6, 150])
@pytest.mark.parametrize("bad", ["inf", "nan", "2^80"])
def test_what_a_row_does_not_see_does_not_matter(rq_ctx, fresh, bad):
    """The last token's scales are no numbers, or far beyond the others': the tokens before it are as ever."""
    b = batch([90], [fresh], 4, 2, 128, 16)
    want = run(rq_ctx, b)
    page, line = int(b["table"][0, (89 + fresh) // 16]), (89 + fresh) % 16
    for plane in (b["cache"].k_scale, b["cache"].v_scale):
        plane[page, :, line] = 2.0**80 if bad == "2^80" else float(bad)
    got = run(rq_ctx, b)
    compare(got[: fresh - 1].contiguous(), {**b, "q": b["q"][: fresh - 1], "starts": [0, fresh - 1], "lengths": [89 + fresh]})
    assert (got[: fresh - 1] - want[: fresh - 1]).abs().max() <= 1e-4


@pytest.mark.parametrize("fresh", [1, 33])
def test_one_large_value_of_zero_scale(rq_ctx, fresh):
    """Scales of zero, a first token that nearly all weight goes to among them."""
    b = batch([200], [fresh], 4, 2, 128, 16)
    page = int(b["table"][0, 0])
    b["cache"].v_scale[page, :, 0] = 0.0
    b["cache"].v_scale[page, :, 5] = 0.0
    b["cache"].k_scale[page, :, 0] *= 4.0
    compare(run(rq_ctx, b), b, norm=None)


def test_rows_past_the_batch_stay_and_the_same_bits_come_back(rq_ctx):
    import torch

    b = batch([500, 3000, 0], [1, 1, 1], 8, 2, 128, 16)
    b["q"] = torch.cat([b["q"], b["q"]])
    y = torch.full(b["q"].shape, 9.0, device="cuda")
    first = run(rq_ctx, b, y=y).clone()
    assert (first[3:] == 9.0).all()
    for _ in range(3):
        assert torch.equal(run(rq_ctx, b, y=y), first)


@pytest.mark.parametrize("fresh,cached", [(1, 20000), (2, 9000), (60, 3000), (300, 700)])
def test_long_caches_over_many_ctas(rq_ctx, fresh, cached):
    import torch

    hq, hk, d = 4, 2, 128
    b = batch([cached], [fresh], hq, hk, d, 64)
    got = run(rq_ctx, b)
    k, v = values(b["cache"], "k"), values(b["cache"], "v")
    n = cached + fresh
    pages = b["table"][0, : ref.pages(n, 64)].long()
    k, v = (x[pages].transpose(0, 1).reshape(hk, -1, d)[:, :n] for x in (k, v))
    q = b["q"].double().reshape(fresh, hk, hq // hk, d)
    score = torch.einsum("thgd,hkd->hgtk", q, k) * d**-0.5
    seen = torch.arange(n, device="cuda")[None] <= cached + torch.arange(fresh, device="cuda")[:, None]
    w = torch.softmax(score.masked_fill(~seen, -torch.inf), -1)
    want = torch.einsum("hgtk,hkd->thgd", w, v).reshape(fresh, hq, d)
    assert (got.double() - want).norm() <= 5e-6 * want.norm()


def test_a_recorded_step_over_codes(rq_ctx):
    """Store and attention recorded together, replayed over other lengths, and on another stream."""
    import torch

    import recipe_dev_b200 as rq

    hq, hk, d, page = 8, 2, 64, 16
    gen = torch.Generator(device="cuda").manual_seed(7)
    cache = rq.KvCache.empty(8, hk, page, d, torch.int8)
    table = torch.tensor([[5, 2, 7]], dtype=torch.int32, device="cuda")
    qkv, q_out, y = torch.empty((1, (hq + 2 * hk) * d), device="cuda"), torch.empty((1, hq * d), device="cuda"), torch.empty((1, hq * d), device="cuda")
    slot, position, starts, length = (torch.zeros(n, dtype=torch.int32, device="cuda") for n in (1, 1, 2, 1))
    starts[1] = 1
    rotation = rq_ctx.rope_table(64, d)
    parts = qkv.split([hq * d, hk * d, hk * d], dim=1)
    rq_ctx.attention_reserve()

    def step(stream=None):
        rq_ctx.rope_store(*parts, position, slot, rotation, cache, q_out=q_out, stream=stream)
        rq_ctx.attention(q_out, cache, table, starts, length, max_fresh=1, y=y, stream=stream)

    step()
    torch.cuda.synchronize()
    step(rq_ctx.sequence_begin())
    sequence = rq_ctx.sequence_end()
    side = torch.cuda.Stream()
    for p in range(40):
        qkv.copy_(torch.randn(qkv.shape, generator=gen, device="cuda"))
        slot.fill_(int(table[0, p // page]) * page + p % page)
        position.fill_(p)
        length.fill_(p + 1)
        if p % 3 == 2:
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                step()
            torch.cuda.current_stream().wait_stream(side)
        else:
            sequence.run()
        torch.cuda.synchronize()
        want, bound = ref.attention(q_out.reshape(1, hq, d), values(cache, "k"), values(cache, "v"), table, [0, 1], [p + 1], d**-0.5)
        assert ((y.double().reshape(1, hq, d) - want).abs() <= bound).all()
    sequence.free()
    rq_ctx.check()


def test_refusals(rq_ctx):
    import torch

    import recipe_dev_b200 as rq

    codes, scales = torch.zeros((2, 2, 16, 128), dtype=torch.int8, device="cuda"), torch.zeros((2, 2, 16), device="cuda")
    for wrong in ((codes, codes), (codes, codes, scales), (codes, codes, scales, scales[:, :1]), (codes, codes, scales.double(), scales.double()), (codes, codes, scales.cpu(), scales.cpu()),
                  (codes.half(), codes.half(), scales, scales), (codes, codes, scales, scales.transpose(0, 1).contiguous().transpose(0, 1))):
        with pytest.raises(ValueError):
            rq.KvCache(*wrong)
    x, i = torch.zeros((4, 256), device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    skewed = torch.zeros(4 * 16 * (128 + 8), dtype=torch.int8, device="cuda").view(2, 2, 16, 136)[..., :128]
    with pytest.raises(rq.RqError, match="multiples of 16"):
        rq_ctx.rope_store(x, x, x, i, i, None, rq.KvCache(skewed, skewed, scales, scales))
    rq_ctx.check()
