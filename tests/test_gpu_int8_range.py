"""Attention over 8-bit codes whose keys and queries lie near the ends of fp32's range, their products well within it. GPU only (-m gpu).

Bounds: serving_reference.attention's. Multiplications by powers of two round nothing while their results are normal numbers; the sum of codes times digits (of queries over the tensor cores: of
16-bit parts) is a number of 1 or more times such a power, and its product with a key's scale is only less than 2^-126 where the score itself is. Where most weights are next to nothing
their own smallest step counts too (few_weights)."""
import pytest

from tests import serving_reference as ref
from tests.test_gpu_int8_cache import batch, compare, run, values

pytestmark = pytest.mark.gpu

# eight rows a key head, sixteen, and more by the tensor cores: one tile of rows, two
FEW = [(4, 2, 64, 1), (4, 2, 128, 1), (4, 2, 256, 3), (4, 2, 128, 7), (8, 2, 64, 4)]
MANY = [(4, 2, 128, 70), (4, 2, 64, 30), (4, 2, 128, 25), (4, 2, 64, 70)]


def sized(hq, hk, d, fresh, q_size, k_size):
    b = batch([100], [fresh], hq, hk, d, 16, seed=fresh)
    b["q"].mul_(q_size)
    b["cache"].k_scale.mul_(k_size)
    return b


def few_weights(got, b, window=0):
    """compare, for rows whose weights times values' scales are nearly all one key's. A weight times its value's scale, x_j = a_j sv_j, is two f16 parts, whose smallest step is 2^-24: off by 2^-25 however small it
    is. Codes times that over the sum of weights, which is at least the top key's, 2^(12 - level) with 2^level <= the largest sv: 2^-37 max sv sum_j |c_j| for each output, beside the bound that is
    relative to the weights' own sum (an element of code zero where all weight goes has next to nothing there)."""
    import torch

    c, keys, hq, d = b["cache"], b["lengths"][0], b["hq"], b["d"]
    hk = c.heads
    want, bound = ref.attention(b["q"].reshape(-1, hq, d), values(c, "k"), values(c, "v"), b["table"], b["starts"], b["lengths"], d**-0.5, window)
    pages = b["table"][0, : ref.pages(keys, 16)].long()
    codes, scales = c.v[pages].transpose(0, 1).reshape(hk, -1, d)[:, :keys], c.v_scale[pages].transpose(0, 1).reshape(hk, -1)[:, :keys]
    step = 2.0**-37 * scales.amax(1, keepdim=True).double() * codes.double().abs().sum(1)
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all() and (off <= bound + step.repeat_interleave(hq // hk, 0)).all()


def opposite(ctx, form, power):
    b = sized(*form, 2.0**-power, 2.0**power)
    compare(run(ctx, b), b)


def keys_of_all_sizes(ctx, form):
    """From 2^-110 to 2^110 in one tile: next to the largest the others are nothing, but for a request whose queries are all the smaller."""
    import torch

    b = sized(*form, 2.0**-107, 1.0)
    gen = torch.Generator(device="cuda").manual_seed(2)
    b["cache"].k_scale.mul_(2.0 ** torch.randint(-110, 111, b["cache"].k_scale.shape, generator=gen, device="cuda"))
    few_weights(run(ctx, b), b)


def queries_of_different_sizes(ctx, form):
    b = sized(*form, 2.0**-103, 2.0**105)
    b["q"][:, ::2] *= 2.0**-9
    b["q"][:, : form[2]] *= 2.0**-20  # (a whole head)
    compare(run(ctx, b), b, norm=None)


def scales_of_scores(ctx, form, scale, q_size, k_size):
    b = sized(*form, q_size, k_size)
    compare(run(ctx, b, scale=scale), b, scale=scale, norm=None)


POWERS = [100, 112, 115, 119, -100, -112, -115, -118]
SCALES = [(2.0**100, 2.0**-53, 2.0**-50), (2.0**-100, 2.0**47, 2.0**50), (3e38, 2.0**-70, 2.0**-61), (2.0**-140, 2.0**40, 2.0**97), (2.0**60, 2.0**30, 2.0**-93), (2.0**20, 2.0**95, 2.0**-118), (2.0**-20, 2.0**-90, 2.0**107)]


@pytest.mark.parametrize("form", FEW)
@pytest.mark.parametrize("power", POWERS)
def test_keys_and_queries_of_opposite_sizes_few_rows(rq_ctx, form, power):
    opposite(rq_ctx, form, power)


@pytest.mark.parametrize("form", FEW)
def test_keys_of_all_sizes_few_rows(rq_ctx, form):
    keys_of_all_sizes(rq_ctx, form)


@pytest.mark.parametrize("form", FEW)
def test_queries_of_different_sizes_few_rows(rq_ctx, form):
    queries_of_different_sizes(rq_ctx, form)


@pytest.mark.parametrize("form", FEW)
@pytest.mark.parametrize("scale,q_size,k_size", SCALES)
def test_scales_of_scores_few_rows(rq_ctx, form, scale, q_size, k_size):
    scales_of_scores(rq_ctx, form, scale, q_size, k_size)


@pytest.mark.parametrize("form", MANY)
@pytest.mark.parametrize("power", POWERS)
def test_keys_and_queries_of_opposite_sizes_many_rows(rq_ctx, form, power):
    opposite(rq_ctx, form, power)


@pytest.mark.parametrize("form", MANY)
def test_keys_of_all_sizes_many_rows(rq_ctx, form):
    keys_of_all_sizes(rq_ctx, form)


@pytest.mark.parametrize("form", MANY)
def test_queries_of_different_sizes_many_rows(rq_ctx, form):
    queries_of_different_sizes(rq_ctx, form)


@pytest.mark.parametrize("form", MANY)
@pytest.mark.parametrize("scale,q_size,k_size", SCALES)
def test_scales_of_scores_many_rows(rq_ctx, form, scale, q_size, k_size):
    scales_of_scores(rq_ctx, form, scale, q_size, k_size)


@pytest.mark.parametrize("form", MANY)
@pytest.mark.parametrize("window", [0, 40])
def test_far_keys_among_usual_ones_many_rows(rq_ctx, form, window):
    """Tiles with keys of far sizes beside tiles without one: of one key head next to nothing, of the other the only ones that its queries tell apart. One value is 2^30 times the others:
    where its code is zero an output is theirs alone, whose weights times scales are f16 numbers of few bits."""
    b = sized(*form, 1.0, 1.0)
    c, d, group = b["cache"], form[2], form[0] // form[1]
    c.k_scale[int(b["table"][0, 1]), 0, 3] *= 2.0**-90
    c.k_scale[int(b["table"][0, 6]), 0, 7] = 0.0
    b["q"][:, group * d :] *= 2.0**-70
    for page, line in ((0, 5), (4, 0), (6, 7)):
        c.k_scale[int(b["table"][0, page]), 1, line] *= 2.0**70
    c.v_scale[int(b["table"][0, 4]), :, 2] *= 2.0**30
    few_weights(run(rq_ctx, b, window=window), b, window)
