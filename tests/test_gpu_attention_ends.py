"""Attention at the ends of the sizes that the header allows: scores of nearly 2^24 over every type of cache, and the smallest and largest values over 8-bit codes. GPU only (-m gpu).

A row's weights are 2^(score - base), score - base one rounding of base away from what it is: 1 at most below 2^24 (2^25 in powers of two), so that an f16 weight, 2^12 at most otherwise, is a number."""
import pytest

from tests import serving_reference as ref
from tests import test_gpu_attention as wide
from tests import test_gpu_int8_cache as codes

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f16", "bf16", "int8"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("fresh", [1, 6, 80])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_of_nearly_2_to_the_24(rq_ctx, dtype, d, fresh, sign):
    """One key is a row's own direction: all weight is its. Or all scores are far below zero, and the least of them counts. Scores in 32 bits are off by 2 d 2^-24 2^24 = 512 at most."""
    import torch

    of, n = (codes if dtype == "int8" else wide), 100 + fresh
    b = of.batch([100], [fresh], 4, 2, d, 16, **({} if dtype == "int8" else dict(dtype=dtype)))
    cache, pages = b["cache"], b["table"][0, : ref.pages(n, 16)].long()

    def flat(name):
        plane = codes.values(cache, name) if dtype == "int8" else getattr(cache, name)
        return plane[pages].transpose(0, 1).reshape(2, -1, d)[:, :n].double()

    if dtype == "int8":
        cache.k_scale[pages] = 1.0 / 64
    if sign < 0:  # one element alone, smaller from token to token: 2 in the cached keys, then from 1 + (fresh - 1) / 128 to 1 (numbers of eight bits)
        cache.k[pages] = 0
        for j in range(n):
            steps = 128 if j < 100 else n - 1 - j
            at = (int(pages[j // 16]), slice(None), j % 16)
            if dtype == "int8":
                cache.k[(*at, 3)], cache.k_scale[at] = 64, (1 + steps / 128) / 64
            else:
                cache.k[(*at, 3)] = 1 + steps / 128
    k, v = flat("k"), flat("v")
    target = k[:, 17]  # (every row sees it)
    q = sign * target / target.square().sum(1, keepdim=True) * 2.0**24 * 0.98
    b["q"].copy_(q.repeat_interleave(2, 0).reshape(1, -1).expand(fresh, -1))
    scores = torch.einsum("thd,hkd->htk", b["q"].double().reshape(fresh, 4, d), k.repeat_interleave(2, 0))
    seen = torch.arange(n, device="cuda")[None] <= 100 + torch.arange(fresh, device="cuda")[:, None]
    best = scores.masked_fill(~seen, -torch.inf).topk(2, dim=2)
    assert scores.abs().max() < 2.0**24 and (best.values[..., 0] - best.values[..., 1]).min() > 1500
    got = of.run(rq_ctx, b, scale=1.0).double()
    want = v.repeat_interleave(2, 0).gather(1, best.indices[..., :1].expand(-1, -1, d)).transpose(0, 1)
    assert torch.isfinite(got).all() and ((got - want).abs() <= 2.0**-18 * want.abs()).all()


@pytest.mark.parametrize("hq,hk,d", [(4, 2, 64), (4, 2, 128), (4, 2, 256)])
@pytest.mark.parametrize("fresh", [1, 6, 80])
@pytest.mark.parametrize("power", [-86, 86])
def test_the_smallest_and_the_largest_values_over_codes(rq_ctx, hq, hk, d, fresh, power):
    b = codes.batch([100], [fresh], hq, hk, d, 16)
    b["cache"].v_scale.mul_(2.0**power)
    largest = codes.values(b["cache"], "v")[b["table"][0, 0]].abs().amax(-1)
    assert largest.min() >= 2.0**-86 and largest.max() <= 2.0**90
    codes.compare(codes.run(rq_ctx, b), b)
