"""Attention whose running maximum stays where it is over many tiles: the sums so far must be carried on as they are, not by a factor that is nearly
one. GPU only (-m gpu).

The bound: a weight is one rounding of its exponent (2^-21 of about 12, ln 2 of which is relative) and an exponential of 2^-22, a score a chain of products in
32 bits, all of them independent from key to key; over ten thousand keys of nearly equal weights what they leave of a head's 2-norm is far
below 2e-6. A factor that is off by one step on every tile would add up to that many steps."""
import pytest

pytestmark = pytest.mark.gpu

PAGE = 64


def queries(kind, shape, gen):
    """Flat heads (no key stands out), or scores that all lie about -5."""
    import torch

    x = torch.randn(shape, generator=gen, device="cuda")
    if kind == "flat":
        return x * torch.linspace(0.3, 0.7, shape[1], device="cuda")[:, None]
    return 0.3 * x - 5.0 * shape[-1] ** -0.5


def served(ctx, kind, dtype, d, hq, hk, keys, requests, fresh, gen_seed=0):
    """requests of `keys` positions each over the same pages in an order of their own, `fresh` new tokens each. The keys' lines lie about 1 + noise (negative
    scores) or about 0 (flat). Returns a function that compares request r of the first n served."""
    import torch

    import recipe_dev_b200 as rq

    gen = torch.Generator(device="cuda").manual_seed(gen_seed)
    kv = {"f16": torch.float16, "bf16": torch.bfloat16}[dtype]
    pages = keys // PAGE
    k, v = (torch.randn((pages, hk, PAGE, d), generator=gen, device="cuda") for _ in range(2))
    if kind != "flat":
        k = 0.3 * k + 1.0
    cache = rq.KvCache(k.to(kv), v.to(kv))
    table = torch.stack([torch.randperm(pages, generator=gen, device="cuda") for _ in range(requests)]).int()
    q = queries(kind, (requests * fresh, hq, d), gen)

    def run(n):
        i32 = dict(dtype=torch.int32, device="cuda")
        y = ctx.attention(q[: n * fresh], cache, table[:n], torch.arange(n + 1, **i32) * fresh, torch.full((n,), keys, **i32), max_fresh=fresh)
        ctx.check()
        return y

    def worst(y, r):
        """The largest relative 2-norm of a head of a token of request r."""
        mine = slice(r * fresh, (r + 1) * fresh)
        at = table[r].long()
        want = torch.empty((fresh, hq, d), dtype=torch.float64, device="cuda")
        position = torch.arange(keys - fresh, keys, device="cuda")
        hidden = torch.arange(keys, device="cuda")[None] > position[:, None]
        for h in range(hk):
            kk, vv = (c[at, h].reshape(keys, d).double() for c in (cache.k, cache.v))
            for g in range(h * (hq // hk), (h + 1) * (hq // hk)):
                want[:, g] = torch.softmax((q[mine, g].double() @ kk.T * d**-0.5).masked_fill(hidden, float("-inf")), 1) @ vv
        return ((y[mine].double() - want).norm(dim=-1) / want.norm(dim=-1)).max().item()

    return run, worst


@pytest.mark.parametrize("kind", ["flat", "negative"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d,hq,hk", [(64, 8, 8), (128, 16, 4), (256, 4, 4)])
def test_one_token_each(rq_ctx, kind, dtype, d, hq, hk):
    """Some hundred to a thousand tiles a warp; a request by itself, dealt out over all CTAs, and among 63 others, alike."""
    run, worst = served(rq_ctx, kind, dtype, d, hq, hk, 32768, 64, 1)
    among, alone = run(64), run(1)
    assert max(worst(among, r) for r in (0, 1, 31, 63)) <= 2e-6
    assert worst(alone, 0) <= 2e-6


@pytest.mark.parametrize("kind", ["flat", "negative"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d,fresh", [(64, 9), (128, 9), (128, 40)])
def test_chunks(rq_ctx, kind, dtype, d, fresh):
    """36 rows a key head (two pipes over alternate tiles of keys) and 160 (f16: two tiles of rows), one or two hundred tiles a CTA and pipe."""
    run, worst = served(rq_ctx, kind, dtype, d, 32, 8, 65536, 12, fresh)
    among, alone = run(12), run(1)
    assert max(worst(among, r) for r in (0, 5, 11)) <= 2e-6
    assert worst(alone, 0) <= 2e-6
