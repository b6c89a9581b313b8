"""The next token against a 64-bit ranking and running sum. GPU only (-m gpu).

The kernel's weights are whole numbers of 2^-40 from fp32 exponentials: a share of the mass is off by less than 2^-20. Random numbers and
top_p are therefore put in the middle of a token's stretch of the running sum, and a token with too short a stretch is not asked for;
the tokens must then be the same, their probabilities within a relative 2^-18."""
import math
import random

import pytest

from tests import serving_reference as ref

pytestmark = pytest.mark.gpu


def draw(ctx, rows, uniform, temperature=None, top_k=None, top_p=None, min_p=None):
    import torch

    def dev(a, kind=torch.float32):
        return None if a is None else torch.tensor(a, dtype=kind, device="cuda")

    x = rows if isinstance(rows, torch.Tensor) else dev(rows)
    n = x.shape[0]
    probability, kept = torch.empty(n, device="cuda"), torch.empty(n, dtype=torch.int32, device="cuda")
    token = ctx.sample(x, dev(uniform), dev(temperature), dev(top_k, torch.int32), dev(top_p), dev(min_p), probability=probability, kept=kept)
    ctx.check()
    return token.tolist(), probability.tolist(), kept.tolist()


def middle(kept, token):
    """A random number in the middle of the token's stretch."""
    return (sum(kept[:token]) + kept[token] / 2) / sum(kept)


def between(weights, order, count):
    """A top_p that keeps the first `count` tokens by rank."""
    total, before = sum(weights), sum(weights[i] for i in order[: count - 1])
    return (before + weights[order[count - 1]] / 2) / total


@pytest.mark.parametrize("vocabulary,rows", [(1, 2), (2, 3), (31, 4), (1000, 8), (1024, 3), (1025, 3), (5003, 6), (32769, 2), (128_256, 2), (262_144, 1), (262_145, 3)])
def test_tokens_of_every_filter(rq_ctx, vocabulary, rows):
    import torch

    rng = random.Random(vocabulary)
    for trial in range(4):
        logits, temperature, top_k, top_p, min_p, uniform, want = [], [], [], [], [], [], []
        for _ in range(rows):
            x = torch.tensor([2.5 * rng.gauss(0, 1) for _ in range(vocabulary)]).tolist()  # the fp32 values
            t = torch.tensor(rng.choice([0.25, 0.7, 1.0, 1.7])).item()
            k = rng.choice([0, 1, 2, 40, 1000, vocabulary, vocabulary + 5]) if trial % 2 else 0
            m = torch.tensor(rng.choice([0.0, 0.03, 0.2])).item() if trial >= 2 else 0.0
            w, order = ref.kept_weights(x, t, k, 1.0, 0.0)
            ranked = [i for i in order if w[i] > 0]
            p = between(w, order, rng.randint(1, min(len(ranked), 300))) if rng.random() < 0.7 else 1.0
            p = torch.tensor(p).item()
            w, _ = ref.kept_weights(x, t, k, p, m)
            total = sum(w)
            heavy = [i for i in range(vocabulary) if w[i] > 2e-5 * total]
            token = rng.choice(heavy)
            logits.append(x), temperature.append(t), top_k.append(k), top_p.append(p), min_p.append(m), uniform.append(middle(w, token))
            want.append((token, w[token] / sum(w), sum(v > 0 for v in w)))
        got = draw(rq_ctx, logits, uniform, temperature, top_k, top_p, min_p)
        for r in range(rows):
            assert got[0][r] == want[r][0], (vocabulary, trial, r)
            assert abs(got[1][r] - want[r][1]) <= 2.0**-18 * want[r][1]
            assert abs(got[2][r] - want[r][2]) <= (0 if top_k[r] or top_p[r] < 1 or min_p[r] else 0.001 * want[r][2])  # (without a filter the last weights are about 2^-40)


def test_no_filters_and_null_parameters(rq_ctx):
    x = [[0.5, 2.0, -1.0, 2.0, 0.0]]
    w, _ = ref.kept_weights(x[0], 1.0, 0, 1.0, 0.0)
    for i in range(5):
        token, probability, kept = draw(rq_ctx, x, [middle(w, i)])
        assert token == [i] and kept == [5] and abs(probability[0] - w[i] / sum(w)) < 1e-6


@pytest.mark.parametrize("vocabulary", [7, 3000, 70_000])
def test_equal_logits_go_by_index(rq_ctx, vocabulary):
    import torch

    x = torch.zeros((1, vocabulary), device="cuda")
    x[0, ::2] = -0.0  # equal to +0
    for k in (1, 3, vocabulary - 1):
        for u, want in ((0.0, 0), (0.999999, k - 1 if k < 50_000 else None)):
            token, _, kept = draw(rq_ctx, x, [u], [1.0], [k])
            assert kept == [k] and (want is None or token == [want])
    token, probability, kept = draw(rq_ctx, x, [0.5], None, None, [2.5 / vocabulary])
    assert kept == [3] and token == [1] and abs(probability[0] - 1 / 3) < 1e-6
    assert draw(rq_ctx, x, [0.9], [0.0])[0] == [0] and draw(rq_ctx, x, [0.9], [1.0], None, [0.0])[0] == [0]  # greedy, and an empty nucleus
    x[0, 5:] = 1.0
    assert draw(rq_ctx, x, [0.9], [0.0]) == ([5], [1.0], [1])
    assert draw(rq_ctx, x, [0.9], [1.0], [1])[0] == [5]


def test_infinities_and_nan(rq_ctx):
    inf, nan = math.inf, math.nan
    x = [[nan, 1.0, -inf, 3.0], [-inf, -inf, nan, -inf], [inf, 0.0, inf, nan], [nan, nan, -1e30, nan], [-inf, 3.4e38, -3.4e38, 0.0]]
    token, probability, kept = draw(rq_ctx, x, [0.99, 0.3, 0.75, 0.5, 0.5])
    assert token == [3, -1, 2, 2, 1] and kept == [2, 0, 2, 1, 1]
    assert probability[1:] == [0.0, 0.5, 1.0, 1.0] and abs(probability[0] - 1 / (1 + math.exp(-2))) < 1e-6
    for t in (0.0, -1.0):
        assert draw(rq_ctx, x, [0.9] * 5, [t] * 5)[0] == [3, -1, 0, 2, 1]
    assert draw(rq_ctx, x, [0.0] * 5, [1e-30] * 5)[0] == [3, -1, 0, 2, 1]


def test_random_numbers_at_the_ends(rq_ctx):
    x = [[0.0, 0.0, 0.0, -50.0]] * 6
    token, _, kept = draw(rq_ctx, x, [0.0, 1.0, -1.0, 2.0, math.nan, 1.0 - 2.0**-24])
    assert token == [0, 2, 0, 2, 0, 2] and kept == [3] * 6  # e^-50 is below 2^-40: no weight


def test_strided_rows_and_the_same_answer_every_time(rq_ctx):
    import torch

    gen = torch.Generator(device="cuda").manual_seed(5)
    plane = 3 * torch.randn((9, 50_007), generator=gen, device="cuda")
    x, u = plane[:, 3:50_004], torch.rand(9, generator=gen, device="cuda")
    p = torch.full((9,), 0.9, device="cuda")
    first = rq_ctx.sample(x, u, top_p=p).tolist()
    assert rq_ctx.sample(x.contiguous(), u, top_p=p).tolist() == first
    assert rq_ctx.sample(x.contiguous().double().float().clone(), u, top_p=p).tolist() == first
    for r in range(9):  # a row by itself
        assert rq_ctx.sample(x[r : r + 1], u[r : r + 1], top_p=p[:1]).tolist() == first[r : r + 1]


def test_many_rows(rq_ctx):
    import torch

    gen = torch.Generator(device="cuda").manual_seed(6)
    x, u = 2 * torch.randn((700, 300), generator=gen, device="cuda"), torch.rand(700, generator=gen, device="cuda")
    got = rq_ctx.sample(x, u, temperature=torch.zeros(700, device="cuda"))
    assert torch.equal(got.long(), x.argmax(1))
    got = rq_ctx.sample(x, u, top_k=torch.ones(700, dtype=torch.int32, device="cuda"))
    assert torch.equal(got.long(), x.argmax(1))


def test_refusals(rq_ctx):
    import torch

    import recipe_dev_b200 as rq

    x, u = torch.zeros((2, 8), device="cuda"), torch.zeros(2, device="cuda")
    with pytest.raises(ValueError):
        rq_ctx.sample(x.half(), u)
    with pytest.raises(ValueError):
        rq_ctx.sample(x, u[:1])
    with pytest.raises(ValueError):
        rq_ctx.sample(x, u, top_k=u)
    with pytest.raises(ValueError):
        rq_ctx.sample(x.t(), torch.zeros(8, device="cuda"))
    wide = torch.zeros((1, (1 << 20) + 1), device="cuda")
    with pytest.raises(rq.RqError, match="at most 1048576"):
        rq_ctx.sample(wide, u[:1])
    assert rq_ctx.sample(wide[:, :-1], u[:1]).tolist() == [0]
    assert rq_ctx.lib.rq_sample(rq_ctx.handle, x.data_ptr(), 4, 2, 8, None, None, None, None, u.data_ptr(), x.data_ptr(), None, None, None) == -1  # rows that overlap
    assert rq_ctx.lib.rq_sample(rq_ctx.handle, None, 8, 2, 8, None, None, None, None, u.data_ptr(), x.data_ptr(), None, None, None) == -1
    rq_ctx.check()
