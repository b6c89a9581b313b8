"""Sampling by filters outside their ranges: they count as the nearest end of it (NaN: no filter). GPU only (-m gpu)."""
import math

import pytest

from tests.test_gpu_sample import draw

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocabulary", [10, 1000, 40_000, 300_000])
@pytest.mark.parametrize("rows", [1, 70])
@pytest.mark.parametrize("top_p", [-0.5, -30.0, -1e30, -math.inf, 0.0])
def test_a_top_p_below_zero_keeps_the_largest(rq_ctx, vocabulary, rows, top_p):
    import torch

    gen = torch.Generator(device="cuda").manual_seed(vocabulary)
    x = 2 * torch.randn((rows, vocabulary), generator=gen, device="cuda")
    best = x.argmax(1).tolist()
    assert draw(rq_ctx, x, [0.999] * rows, [0.9] * rows, None, [top_p] * rows) == (best, [1.0] * rows, [1] * rows)
    assert draw(rq_ctx, x, [0.999] * rows, [1e-3] * rows, [600] * rows, [top_p] * rows, [0.5] * rows) == (best, [1.0] * rows, [1] * rows)


@pytest.mark.parametrize("top_k", [0, 5, 700])
@pytest.mark.parametrize("vocabulary", [10, 3000])
def test_filters_that_are_no_numbers_filter_nothing(rq_ctx, top_k, vocabulary):
    import torch

    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((3, vocabulary), generator=gen, device="cuda")
    u = [0.1, 0.5, 0.97]
    want = draw(rq_ctx, x, u, None, [top_k] * 3)
    assert want[2] == [min(top_k or vocabulary, vocabulary)] * 3
    for top_p in (math.nan, 1.0, 7.0, math.inf):
        for min_p in (math.nan, 0.0, -1.0, -math.inf):
            assert draw(rq_ctx, x, u, None, [top_k] * 3, [top_p] * 3, [min_p] * 3) == want


def test_a_min_p_above_one_keeps_the_largest(rq_ctx):
    x = [[0.0, 2.0, 1.0, 2.0]]
    for top_k in (0, 3):
        for min_p in (1.5, math.inf):
            assert draw(rq_ctx, x, [0.9], None, [top_k], None, [min_p]) == ([3], [0.5], [2])
