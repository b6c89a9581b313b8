"""Attention over 8-bit codes: what a batch may look like at its edges. GPU only (-m gpu).

Bounds: test_gpu_int8_cache.py's."""
import pytest

from tests import serving_reference as ref
from tests.test_gpu_int8_cache import batch, compare, run, values

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("max_fresh", [0, 1, 3, 10**9])
@pytest.mark.parametrize("fresh", [[1, 1, 1], [5, 1, 60], [40, 40, 40]])
@pytest.mark.parametrize("hq,hk,d", [(8, 2, 64), (4, 4, 128), (2, 2, 256)])
def test_what_the_host_knows_of_the_longest_request(rq_ctx, max_fresh, fresh, hq, hk, d):
    """Nothing, too little, or too much: only the choice of kernel follows from it."""
    b = batch([70, 0, 33], fresh, hq, hk, d, 16)
    compare(run(rq_ctx, b, max_fresh=max_fresh), b)


@pytest.mark.parametrize("fresh", [9, 70])
@pytest.mark.parametrize("window", [0, 4])
def test_requests_that_are_longer_than_their_lengths(rq_ctx, fresh, window):
    """Tokens in front of position zero see nothing."""
    b = batch([0, 20], [fresh, fresh], 4, 2, 128, 16)
    b["lengths"][0] = 5
    got = run(rq_ctx, b, window=window)
    assert (got[: fresh - 5] == 0).all()
    compare(got, b, window=window)


@pytest.mark.parametrize("fresh", [1, 50])
def test_tokens_in_front_of_the_first_request_stay(rq_ctx, fresh):
    import torch

    b = batch([90, 17], [fresh, fresh], 4, 2, 64, 16)
    before = 3
    want, bound = ref.attention(b["q"].reshape(-1, 4, 64), values(b["cache"], "k"), values(b["cache"], "v"), b["table"], b["starts"], b["lengths"], 64**-0.5)
    b["q"] = torch.cat([torch.full((before, 4 * 64), float("nan"), device="cuda"), b["q"], b["q"][:1]])
    b["starts"] = [s + before for s in b["starts"]]
    got = run(rq_ctx, b)
    assert (got[:before] == 9.0).all() and (got[before + 2 * fresh :] == 9.0).all()
    assert ((got[before : before + 2 * fresh].double() - want).abs() <= bound).all()


@pytest.mark.parametrize("max_fresh", [1, 200])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_a_batch_without_a_token(rq_ctx, max_fresh, d):
    b = batch([30, 40], [1, 1], 4, 2, d, 16)
    b["starts"] = [0, 0, 0]
    assert (run(rq_ctx, b, max_fresh=max_fresh) == 9.0).all()


@pytest.mark.parametrize("fresh", [1, 13])
def test_the_most_requests(rq_ctx, fresh):
    """4096: one more fits no call. 13 tokens of four heads a key head go to the tensor cores."""
    cached = [(37 * r) % 23 for r in range(4096)]
    b = batch(cached, [fresh] * 4096, 4, 1, 64, 8)
    got = run(rq_ctx, b)
    for r in (0, 1, 1000, 2047, 2048, 4094, 4095):
        mine = slice(r * fresh, (r + 1) * fresh)
        compare(got[mine].contiguous(), dict(b, q=b["q"][mine], table=b["table"][r : r + 1], starts=[0, fresh], lengths=[cached[r] + fresh]), norm=None)


@pytest.mark.parametrize("fresh,d", [(1, 64), (1, 128), (2, 256), (40, 64), (70, 128)])
def test_two_requests_over_the_same_pages(rq_ctx, fresh, d):
    b = batch([100, 100], [fresh, fresh], 4, 2, d, 16)
    b["table"][1, :6] = b["table"][0, :6]  # (a prompt's beginning that both share)
    compare(run(rq_ctx, b), b)


@pytest.mark.parametrize("fresh", [1, 70])
def test_a_cache_past_2_to_the_32_bytes(rq_ctx, fresh):
    """Pages at the end of five billion codes and a page in front: the store writes them, attention reads them."""
    import torch

    import recipe_dev_b200 as rq

    hq, hk, d, page, pages = 8, 8, 128, 128, 38200
    cache = rq.KvCache.empty(pages, hk, page, d, torch.int8)
    assert cache.k.numel() > 2**32 + 2**29
    gen = torch.Generator(device="cuda").manual_seed(1)
    n = 300 + fresh
    mine = [pages - 1, 3, pages - 2, pages - 5][: ref.pages(n, page)]
    table = torch.tensor([mine], dtype=torch.int32, device="cuda")
    at = torch.arange(n, device="cuda")
    slots = (table[0].long()[at // page] * page + at % page).int()
    q, k, v = (torch.randn((n, h * d), generator=gen, device="cuda") for h in (hq, hk, hk))
    rq_ctx.rope_store(q, k, v, at.int(), slots, None, cache)
    for x, name in ((k, "k"), (v, "v")):
        step = x.view(n, hk, d).abs().amax(-1, keepdim=True).double() / 127
        held = values(rq.KvCache(cache.k[mine], cache.v[mine], cache.k_scale[mine], cache.v_scale[mine]), name).transpose(1, 2).reshape(-1, hk, d)[:n]
        assert ((held - x.view(n, hk, d).double()).abs() <= 0.501 * step).all()
    few = rq.KvCache(*(a[mine].contiguous() for a in (cache.k, cache.v, cache.k_scale, cache.v_scale)))
    b = dict(q=q[:fresh], cache=cache, table=table, starts=[0, fresh], lengths=[n], hq=hq, d=d)
    got = run(rq_ctx, b)
    compare(got, dict(b, cache=few, table=torch.arange(len(mine), dtype=torch.int32, device="cuda")[None]))
