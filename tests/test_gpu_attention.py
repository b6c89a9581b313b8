"""Attention of new tokens over the paged cache against 64 bits, at the sizes and masks where it can go wrong. GPU only (-m gpu).

The bound of each output is derived beside the reference (serving_reference.attention); over a whole call the outputs, fp32 sums over
fp32 queries, are also within 5e-6 in the 2-norm."""
import random

import pytest

from tests import serving_reference as ref

pytestmark = pytest.mark.gpu


def batch(cached, fresh, hq, hk, d, page, dtype="f16", seed=0, spread=2.0, order="heads", width=0, offset=0, pad=0):
    """A batch over randomly placed pages; every position past a request's length, and every page that nobody owns, holds NaN."""
    import torch

    import recipe_dev_b200 as rq

    kind = {"f16": torch.float16, "bf16": torch.bfloat16}[dtype]
    gen = torch.Generator(device="cuda").manual_seed(seed)
    lengths = [c + f for c, f in zip(cached, fresh)]
    held = [ref.pages(n, page) for n in lengths]
    total = sum(held) + 2
    shape = (total, hk, page, d) if order == "heads" else (total, page, hk, d)
    k, v = (torch.full(shape, float("nan"), dtype=kind, device="cuda") for _ in range(2))
    cache = rq.KvCache(k, v) if order == "heads" else rq.KvCache(k.transpose(1, 2), v.transpose(1, 2))
    ids = random.Random(seed).sample(range(total), sum(held))
    width = width or max(max(held), 1) + 1
    table = torch.full((len(cached), width + 3), 2**30, dtype=torch.int32, device="cuda")[:, :width]
    for r, n in enumerate(lengths):
        mine = [ids.pop() for _ in range(held[r])]
        for i, page_id in enumerate(mine[:width]):
            table[r, i] = page_id
        for i, page_id in enumerate(mine):
            lines = min(page, n - i * page)
            cache.k[page_id, :, :lines] = torch.randn((hk, lines, d), generator=gen, device="cuda").to(kind)
            cache.v[page_id, :, :lines] = torch.randn((hk, lines, d), generator=gen, device="cuda").to(kind)
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


def compare(got, b, window=0, scale=None):
    import torch

    want, bound = ref.attention(b["q"].reshape(-1, b["hq"], b["d"]), b["cache"].k, b["cache"].v, b["table"], b["starts"], b["lengths"], scale or b["d"] ** -0.5, window)
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all() and (off <= bound).all(), float((off - bound).max())
    assert off.norm() <= 5e-6 * want.norm()


@pytest.mark.parametrize("hq,hk,d", [(1, 1, 64), (8, 2, 128), (32, 8, 128), (4, 4, 256), (7, 1, 64), (20, 1, 128), (28, 4, 128), (40, 2, 64), (16, 1, 256), (128, 1, 64)])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_one_token_each(rq_ctx, hq, hk, d, dtype):
    b = batch([0, 1, 30, 299, 64, 127], [1] * 6, hq, hk, d, 16, dtype)
    compare(run(rq_ctx, b), b)


@pytest.mark.parametrize("hq,hk,d", [(8, 2, 128), (2, 2, 64), (6, 2, 256), (9, 3, 64), (24, 1, 128)])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_chunks_over_a_cache(rq_ctx, hq, hk, d, dtype):
    b = batch([0, 5, 130, 40, 0], [33, 1, 70, 0, 129], hq, hk, d, 16, dtype)
    compare(run(rq_ctx, b), b)


@pytest.mark.parametrize("page", [1, 2, 8, 32, 64, 128, 256, 4096])
@pytest.mark.parametrize("fresh", [1, 3, 65])
def test_page_sizes(rq_ctx, page, fresh):
    b = batch([200, 0, 77], [fresh] * 3, 8, 2, 128, page)
    compare(run(rq_ctx, b), b)


@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 191, 192, 193, 255, 256, 257, 383, 385])
def test_lengths_about_tile_ends(rq_ctx, length):
    for fresh in {1, min(length, 2), length}:
        b = batch([length - fresh], [fresh], 4, 2, 64, 16, seed=length)
        compare(run(rq_ctx, b), b)


@pytest.mark.parametrize("window", [1, 2, 17, 64, 100, 128, 1000])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_windows(rq_ctx, window, dtype):
    b = batch([0, 300, 63, 500], [40, 1, 130, 5], 4, 2, 128, 16, dtype)
    compare(run(rq_ctx, b, window=window), b, window=window)


@pytest.mark.parametrize("order,offset,pad", [("lines", 0, 0), ("heads", 1, 0), ("lines", 2, 5), ("heads", 4, 4)])
@pytest.mark.parametrize("fresh", [1, 40])
def test_layouts_alignment_and_strides(rq_ctx, order, offset, pad, fresh):
    import torch

    b = batch([60, 3], [fresh, fresh], 6, 2, 128, 16, order=order, offset=offset, pad=pad)
    tokens = b["q"].shape[0]
    plane = torch.full((tokens * (6 * 128 + 7) + 1,), 5.0, device="cuda")
    y = plane[1:].view(tokens, 6 * 128 + 7)[:, : 6 * 128]
    compare(run(rq_ctx, b, y=y), b)
    assert (plane[1:].view(tokens, -1)[:, 6 * 128 :] == 5.0).all() and plane[0] == 5.0


def test_the_host_may_be_wrong_about_the_longest_chunk(rq_ctx):
    """max_fresh chooses a kernel; every kernel serves every batch."""
    b = batch([100, 0, 10], [90, 1, 7], 8, 2, 128, 16)
    for guess in (0, 1, 2, 16, 1000):
        compare(run(rq_ctx, b, max_fresh=guess), b)
    b = batch([100, 20, 10], [1, 1, 1], 8, 2, 128, 16)
    for guess in (0, 1, 1000):
        compare(run(rq_ctx, b, max_fresh=guess), b)


def test_rows_that_see_nothing_get_zeros(rq_ctx):
    """Lengths below the new tokens (earlier rows lie before position 0), pages outside the cache, a table that ends early."""
    import torch

    for fresh in (4, 50):
        b = batch([20, 20, 20], [fresh] * 3, 4, 2, 64, 16)
        b["lengths"][0] = fresh // 2
        b["lengths"][1] = 0
        b["table"][2, 0] = -1
        b["table"][2, 1] = 2**31 - 1
        got = run(rq_ctx, b)
        compare(got, b)
        assert (got[: fresh - fresh // 2] == 0).all() and (got[fresh : 2 * fresh] == 0).all()
    b = batch([300], [2], 4, 2, 64, 16, width=5)  # the table names the first 80 positions only
    compare(run(rq_ctx, b), b)
    b = batch([300], [2], 4, 2, 64, 16)
    b["table"][:] = -1
    assert (run(rq_ctx, b) == 0).all()
    b["lengths"] = [-5]
    assert torch.equal(run(rq_ctx, b), torch.zeros_like(b["q"]).reshape(-1, 4, 64))


def test_tokens_past_the_batch_are_not_written(rq_ctx):
    import torch

    for fresh in (1, 30):
        b = batch([20, 40], [fresh, fresh], 4, 2, 64, 16)
        b["q"] = torch.cat([b["q"], b["q"][:5] * float("nan")])
        got = run(rq_ctx, b)
        assert (got[2 * fresh :] == 9.0).all()
        b["q"], got = b["q"][: 2 * fresh], got[: 2 * fresh]
        compare(got, b)


@pytest.mark.parametrize("fresh,given", [([1, 1, 1], 2), ([3, 40], 30), ([3, 40], 2), ([90, 100], 120), ([4, 5], 4)])
def test_a_batch_longer_than_the_call(rq_ctx, fresh, given):
    """The plan may count more tokens than the arrays that the call is given have room for: those are passed over, the others are what they are."""
    import torch

    b = batch([20] * len(fresh), fresh, 4, 2, 128, 16)
    whole = torch.full(b["q"].shape, 9.0, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    rq_ctx.attention(b["q"][:given], b["cache"], b["table"], torch.tensor(b["starts"], **i32), torch.tensor(b["lengths"], **i32), max_fresh=max(fresh), y=whole[:given])
    rq_ctx.check()
    assert (whole[given:] == 9.0).all()
    want, bound = ref.attention(b["q"].reshape(-1, 4, 128), b["cache"].k, b["cache"].v, b["table"], b["starts"], b["lengths"], 128**-0.5)
    assert ((whole.reshape(-1, 4, 128).double() - want).abs() <= bound)[:given].all()


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf"), -65504.0, 65504.0])
@pytest.mark.parametrize("fresh", [1, 2, 40, 200])
def test_whatever_masked_places_hold(rq_ctx, value, fresh):
    """A key or value that a row does not see has no part in it: a later token's, one left of the window, one past the length."""
    import torch

    b = batch([150], [fresh], 4, 2, 128, 16)
    clean = run(rq_ctx, b, window=64).clone()
    page_of = b["table"][0].tolist()
    for j in (0, 3, 80, 150 - 64, 150 + fresh):  # left of every row's window (or in the last page, past the end)
        if j < 150 + fresh or j % 16:
            b["cache"].k[page_of[j // 16], :, j % 16] = value
            b["cache"].v[page_of[j // 16], :, j % 16] = value
    assert torch.equal(run(rq_ctx, b, window=64), clean)
    if fresh > 1:
        last = 150 + fresh - 1  # the last token's key and value: no row before it sees them
        b["cache"].k[page_of[last // 16], :, last % 16] = value
        b["cache"].v[page_of[last // 16], :, last % 16] = value
        got = run(rq_ctx, b, window=64)
        assert torch.equal(got[:-1], clean[:-1])


def test_scores_far_apart_and_equal(rq_ctx):
    """One key above all others by hundreds, scores that fall and rise along the cache, and keys that are all the same."""
    import torch

    for fresh in (1, 60):
        b = batch([400], [fresh], 4, 2, 64, 16)
        b["q"] *= 40.0
        compare(run(rq_ctx, b), b)
        b["cache"].k[:] = 1.0
        compare(run(rq_ctx, b), b)
        ramp = torch.linspace(-3, 3, 16, device="cuda")[:, None].half()
        for i, page_id in enumerate(b["table"][0].tolist()[:25]):
            b["cache"].k[page_id] = ramp * (i - 12)
        compare(run(rq_ctx, b), b)
        compare(run(rq_ctx, b, scale=1e-30), b, scale=1e-30)


def test_long_contexts_are_the_same_when_dealt_out(rq_ctx):
    """One sequence over many CTAs against 64 bits, and the same bits on every run."""
    import torch

    b = batch([20_000], [1], 8, 2, 128, 64)
    first = run(rq_ctx, b).clone()
    compare(first, b)
    for _ in range(3):
        assert torch.equal(run(rq_ctx, b), first)
    b = batch([9000, 3], [3, 64], 8, 2, 128, 16)
    first = run(rq_ctx, b).clone()
    compare(first, b)
    for _ in range(3):
        assert torch.equal(run(rq_ctx, b), first)


def test_a_cache_beyond_32_bit_offsets(rq_ctx):
    """Element offsets above 2^32: the last pages of an 8.6 GB cache."""
    import torch

    import recipe_dev_b200 as rq

    pages = (2**32 + 2**26) // (8 * 16 * 128)
    plane = torch.empty((pages, 8, 16, 128), dtype=torch.float16, device="cuda")
    cache = rq.KvCache(plane, plane)
    for fresh in (1, 40):
        b = batch([100], [fresh], 8, 8, 128, 16)
        n = ref.pages(100 + fresh, 16)
        for i in range(n):
            plane[pages - 1 - i] = b["cache"].k[b["table"][0, i]]
            b["table"][0, i] = pages - 1 - i
        b["cache"] = cache
        compare(run(rq_ctx, b), b)
    x = torch.randn((1, 8 * 128), device="cuda")
    slot = torch.tensor([pages * 16 - 3], dtype=torch.int32, device="cuda")
    rq_ctx.rope_store(x, x, x, slot, slot, None, cache)
    assert torch.equal(plane[pages - 1, :, 13], x.view(8, 128).half())
    rq_ctx.check()


def test_many_requests(rq_ctx):
    rng = random.Random(4)
    cached = [rng.randint(0, 40) for _ in range(700)]
    fresh = [rng.choice([0, 1, 1, 1, 2]) for _ in range(700)]
    b = batch(cached, fresh, 4, 1, 64, 8)
    compare(run(rq_ctx, b), b)


@pytest.mark.parametrize("hq,hk,d", [(8, 2, 128), (7, 1, 64), (20, 1, 128), (40, 1, 64), (4, 2, 256)])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("cached,fresh", [([40, 700, 0, 5, 300], [1, 1, 150, 0, 1]), ([0, 130, 0], [3, 90, 1]), ([900, 0, 31], [1, 33, 0])])
def test_decode_steps_among_prompts(rq_ctx, hq, hk, d, dtype, cached, fresh):
    b = batch(cached, fresh, hq, hk, d, 16, dtype)
    compare(run(rq_ctx, b), b)
    assert (run(rq_ctx, b) == run(rq_ctx, b)).all()


def test_nothing_but_decode_steps_when_the_host_does_not_know(rq_ctx):
    b = batch([40, 700, 0, 5, 300, 64, 63, 1, 999], [1] * 9, 8, 2, 128, 16)
    compare(run(rq_ctx, b, max_fresh=0), b)
    compare(run(rq_ctx, b, max_fresh=500), b)


@pytest.mark.parametrize("fresh", [[1, 1], [1, 80]])
def test_recorded_and_replayed_over_longer_requests(fresh):
    """The lengths are read when a recorded call runs, not when it is recorded; the work area has to be there before."""
    import torch

    import recipe_dev_b200 as rq

    ctx = rq.Context(0)  # one that has no work area yet
    long = batch([700, 333], fresh, 8, 2, 128, 16)
    starts = torch.tensor(long["starts"], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([30 + fresh[0], 20 + fresh[1]], dtype=torch.int32, device="cuda")
    y = torch.zeros_like(long["q"])
    stream = ctx.sequence_begin()
    with pytest.raises(rq.RqError, match="rq_attention_reserve"):
        ctx.attention(long["q"], long["cache"], long["table"], starts, lengths, max_fresh=max(fresh), y=y, stream=stream)
    ctx.sequence_end().free()
    ctx.attention_reserve()
    stream = ctx.sequence_begin()
    ctx.attention(long["q"], long["cache"], long["table"], starts, lengths, max_fresh=max(fresh), y=y, stream=stream)
    sequence = ctx.sequence_end()
    for now in ([30 + fresh[0], 20 + fresh[1]], long["lengths"]):
        lengths.copy_(torch.tensor(now, dtype=torch.int32))
        sequence.run()
        torch.cuda.synchronize()
        compare(y.reshape(-1, 8, 128), dict(long, lengths=now))
    sequence.free()
    ctx.check()
    ctx.close()


def test_two_streams_share_the_work_area(rq_ctx):
    import torch

    a, b = batch([5000], [1], 8, 2, 128, 16, seed=1), batch([7000, 10], [1, 1], 8, 2, 128, 16, seed=2)
    want = [run(rq_ctx, x).clone() for x in (a, b)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = []
    for _ in range(5):
        for s, x in zip(streams, (a, b)):
            with torch.cuda.stream(s):
                starts, lengths = (torch.tensor(x[k], dtype=torch.int32, device="cuda") for k in ("starts", "lengths"))
                outs.append(rq_ctx.attention(x["q"], x["cache"], x["table"], starts, lengths, max_fresh=1))
    torch.cuda.synchronize()
    for i, y in enumerate(outs):
        assert torch.equal(y.reshape(want[i % 2].shape), want[i % 2])
    rq_ctx.check()


def test_refusals(rq_ctx):
    import torch

    import recipe_dev_b200 as rq

    b = batch([20], [2], 4, 2, 64, 16)
    i = torch.tensor([0, 2], dtype=torch.int32, device="cuda")
    n = torch.tensor([22], dtype=torch.int32, device="cuda")
    with pytest.raises(rq.RqError, match="multiple of the cache"):
        rq_ctx.attention(b["q"][:, :192], b["cache"], b["table"], i, n)
    with pytest.raises(ValueError):
        rq_ctx.attention(b["q"][:, :200], b["cache"], b["table"], i, n)
    with pytest.raises(ValueError):
        rq_ctx.attention(b["q"].half(), b["cache"], b["table"], i, n)
    with pytest.raises(ValueError):
        rq_ctx.attention(b["q"], b["cache"], b["table"], i[:1], n)
    with pytest.raises(ValueError):
        rq_ctx.attention(b["q"], b["cache"], b["table"].long(), i, n)
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(rq.RqError, match="scale"):
            rq_ctx.attention(b["q"], b["cache"], b["table"], i, n, scale=scale)
    with pytest.raises(rq.RqError, match="window"):
        rq_ctx.attention(b["q"], b["cache"], b["table"], i, n, window=-1)
    wide = rq.KvCache.empty(2, 1, 16, 64)
    with pytest.raises(rq.RqError, match="at most 128"):
        rq_ctx.attention(torch.zeros((2, 129 * 64), device="cuda"), wide, b["table"], i, n)
    with pytest.raises(rq.RqError, match="64, 128 or 256"):
        rq_ctx.attention(torch.zeros((2, 96), device="cuda"), rq.KvCache.empty(2, 1, 16, 96), b["table"], i, n)
    rq_ctx.check()
