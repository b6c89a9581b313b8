"""Log probabilities with entropy, rank and alternatives against 64 bits. GPU only (-m gpu).

Bounds. With M = max x, z_i = x_i - M (one rounding), e_i is off by three roundings of z_i and the exponential's two steps, 2^-24 (3 |z_i| + 4) of it; the sum over a row
adds at most 128 roundings (sixteen logits, up to 64 rounds, trees). So log Z is off by 2^-24 (132 + 3 m1 + 2 log Z), m1 = E|z|; a log probability by that and two roundings of z
and itself; the mean of z by 2^-24 (3 m2 + 136 m1) and m1 times the sum's."""
import math

import pytest

pytestmark = pytest.mark.gpu
STEP = 2.0**-24


def run(ctx, logits, token=None, top=0, entropy=True):
    import torch

    rows = logits.shape[0]
    out = dict(entropy=torch.full((rows,), 5.0, device="cuda") if entropy else None)
    if token is not None:
        out.update(logprob=torch.full((rows,), 5.0, device="cuda"), rank=torch.full((rows,), 5, dtype=torch.int32, device="cuda"))
    if top:
        out.update(top_token=torch.full((rows, top), 5, dtype=torch.int32, device="cuda"), top_logprob=torch.full((rows, top), 5.0, device="cuda"))
    got = ctx.logprobs(logits, token, **out)
    ctx.check()
    assert got is out.get("logprob")
    return out


def compare(ctx, logits, token, top):
    import torch

    out = run(ctx, logits, token, top)
    x = torch.where(torch.isnan(logits), -torch.inf, logits).double()
    rows, vocabulary = x.shape
    largest = x.amax(1, keepdim=True)
    z = (x - largest).clamp(min=-1e100)  # (of weight zero: its square has to stay a number)
    p = torch.softmax(x, 1)
    log_sum = torch.logsumexp(z, 1)
    logp = x - largest - log_sum[:, None]
    m1, m2 = (p * z.abs()).sum(1), (p * z.square()).sum(1)
    entropy = log_sum + m1
    of_sum = STEP * (132 + 3 * m1 + 2 * log_sum)
    assert ((out["entropy"].double() - entropy).abs() <= of_sum + STEP * (3 * m2 + 136 * m1 + 2 * entropy) + m1 * of_sum + 1e-30).all()
    inside = (token >= 0) & (token < vocabulary)
    t = token.long().clamp(0, vocabulary - 1)[:, None]
    want = torch.where(inside, logp.gather(1, t)[:, 0], 0.0)
    off = (out["logprob"].double() - want).abs()
    assert torch.where(torch.isinf(want), out["logprob"] == want, off <= of_sum + STEP * 4 * want.abs() + STEP * 2 * log_sum).all()
    index = torch.arange(vocabulary, device="cuda")[None]
    mine = x.gather(1, t)
    rank = ((x > mine) | ((x == mine) & (index < t))).sum(1)
    assert torch.equal(out["rank"].long(), torch.where(inside, rank, -1))
    if top:
        order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top]
        if order.shape[1] < top:
            order = torch.nn.functional.pad(order, (0, top - order.shape[1]), value=-1)
        best = torch.where(order >= 0, logp.gather(1, order.clamp(min=0)), -torch.inf)
        order = torch.where(torch.isinf(best), -1, order)
        assert torch.equal(out["top_token"].long(), order)
        off = (out["top_logprob"].double() - best).abs()
        assert torch.where(torch.isinf(best), out["top_logprob"] == best, off <= of_sum[:, None] + STEP * 4 * best.abs() + STEP * 2 * log_sum[:, None]).all()


def some(rows, vocabulary, seed=0, spread=2.5, offset=0, pad=0):
    import torch

    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = spread * torch.randn(rows * (vocabulary + pad) + offset, generator=gen, device="cuda")[offset:].view(rows, vocabulary + pad)[:, :vocabulary]
    return x, torch.randint(0, vocabulary, (rows,), generator=gen, device="cuda").int()


@pytest.mark.parametrize("vocabulary", [1, 2, 3, 5, 31, 64, 255, 1000, 4095, 4096, 4097, 8191, 32000, 50257, 131073, 262144])
@pytest.mark.parametrize("top", [0, 1, 20, 64])
def test_vocabularies(rq_ctx, vocabulary, top):
    compare(rq_ctx, *some(3, vocabulary, vocabulary), top)


@pytest.mark.parametrize("rows", [1, 2, 5, 37, 64, 150, 700])
@pytest.mark.parametrize("vocabulary", [5000, 40001])
def test_rows(rq_ctx, rows, vocabulary):
    compare(rq_ctx, *some(rows, vocabulary, rows), 20)


def test_the_largest_vocabulary(rq_ctx):
    compare(rq_ctx, *some(2, 1048576), 33)


@pytest.mark.parametrize("offset,pad", [(0, 1), (1, 0), (2, 3), (3, 2), (0, 4)])
@pytest.mark.parametrize("vocabulary", [3, 999, 30001])
def test_alignment_and_strides(rq_ctx, offset, pad, vocabulary):
    compare(rq_ctx, *some(9, vocabulary, offset=offset, pad=pad), 5)


@pytest.mark.parametrize("vocabulary", [700, 20000, 262144])
@pytest.mark.parametrize("top", [1, 20, 64])
@pytest.mark.parametrize("order", ["rising", "falling", "equal", "few values", "two sizes", "late"])
def test_orders_and_ties(rq_ctx, vocabulary, top, order):
    import torch

    x, token = some(2, vocabulary, 4)
    if order in ("rising", "falling"):
        x = torch.sort(x, dim=1, descending=order == "falling").values.contiguous()
    elif order == "equal":
        x.fill_(-3.25)
    elif order == "few values":
        x = torch.round(x)
        x[x == 0] = -0.0
        x[:, ::3] += 0.0
    elif order == "two sizes":
        x = torch.where(x > 0, 1.0, 0.0)
    else:
        x[:, : vocabulary // 2] -= 100.0
    compare(rq_ctx, x, token, top)


@pytest.mark.parametrize("vocabulary", [90, 6000, 150001])
def test_masked_logits(rq_ctx, vocabulary):
    """Logits of -inf, of the type's lowest value, and NaN; a given token among them, and at the ends; rows with fewer numbers than alternatives."""
    import torch

    x, token = some(12, vocabulary, 8)
    lowest = torch.finfo(torch.float32).min
    x[0, ::2], x[1, ::2], x[2, ::3] = -torch.inf, lowest, float("nan")
    x[3, 7:], x[4, :-5], x[5] = -torch.inf, float("nan"), lowest
    x[6, vocabulary // 3 :: 2] = -torch.inf
    for r, t in enumerate((2, 4, 6, 8, 0, vocabulary - 1, vocabulary // 3 + 2, 0, vocabulary - 1, -1, vocabulary, 2**31 - 1)):
        token[r] = t
    compare(rq_ctx, x, token, 20)


def test_rows_without_any_number(rq_ctx):
    import torch

    x = torch.full((3, 5000), -torch.inf, device="cuda")
    x[1] = float("nan")
    x[2, 17] = 3.0
    out = run(rq_ctx, x, torch.tensor([1, 2, 17], dtype=torch.int32, device="cuda"), 3)
    assert out["logprob"].tolist() == [-math.inf, -math.inf, 0.0] and out["rank"].tolist() == [-1, -1, 0] and out["entropy"].tolist() == [0.0, 0.0, 0.0]
    assert out["top_token"].tolist() == [[-1] * 3, [-1] * 3, [17, -1, -1]] and out["top_logprob"].tolist() == [[-math.inf] * 3, [-math.inf] * 3, [0.0, -math.inf, -math.inf]]


@pytest.mark.parametrize("size", [1e-30, 1e-3, 100.0, 1e30])
def test_sizes(rq_ctx, size):
    x, token = some(4, 9000, 2)
    compare(rq_ctx, x * size, token, 7)


def test_far_apart(rq_ctx):
    import torch

    x, token = some(3, 12345, 6)
    x[0, 100], x[1, 12000], x[2] = 300.0, 3e38, -3e38
    compare(rq_ctx, x, token, 4)


def test_the_same_bits_for_a_row_by_itself(rq_ctx):
    import torch

    x, token = some(6, 70000, 9)
    first = run(rq_ctx, x, token, 20)
    again = run(rq_ctx, x, token, 20)
    for name, a in first.items():
        assert torch.equal(a, again[name])


def test_outputs_that_are_not_wanted(rq_ctx):
    import torch

    x, token = some(4, 30000, 5)
    full = run(rq_ctx, x, token, 9)
    assert torch.equal(rq_ctx.logprobs(x, token), full["logprob"])
    alone = torch.empty((4, 9), dtype=torch.int32, device="cuda")
    assert rq_ctx.logprobs(x, top_token=alone) is None and torch.equal(alone, full["top_token"])
    entropy = torch.empty(4, device="cuda")
    rq_ctx.logprobs(x, entropy=entropy)
    assert torch.allclose(entropy, full["entropy"], rtol=1e-5)


def test_recorded_and_on_another_stream(rq_ctx):
    import torch

    x, token = some(3, 65000, 1)
    out = dict(logprob=torch.empty(3, device="cuda"), top_token=torch.empty((3, 5), dtype=torch.int32, device="cuda"))
    rq_ctx.logprobs(x, token, **out)
    torch.cuda.synchronize()
    rq_ctx.logprobs(x, token, **out, stream=rq_ctx.sequence_begin())
    sequence = rq_ctx.sequence_end()
    side = torch.cuda.Stream()
    for seed in range(3):
        fresh, _ = some(3, 65000, 20 + seed)
        x.copy_(fresh)
        sequence.run()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            want = run(rq_ctx, x, token, 5)
        torch.cuda.synchronize()
        assert torch.equal(out["logprob"], want["logprob"]) and torch.equal(out["top_token"], want["top_token"])
    sequence.free()


def test_refusals(rq_ctx):
    import torch

    x, t = torch.zeros((3, 50), device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    f = torch.zeros(3, device="cuda")
    tops = torch.zeros((3, 4), dtype=torch.int32, device="cuda")
    for wrong in (dict(logits=x.double()), dict(logits=x.T), dict(logits=x.cpu()), dict(token=t.long()), dict(token=t[:2]), dict(logprob=f.double()), dict(rank=f), dict(entropy=f[:2]),
                  dict(top_token=tops, top_logprob=torch.zeros((3, 5), device="cuda")), dict(top_token=tops[:2]), dict(top_token=tops[:, :0]), dict(token=None, rank=t), dict(token=None, logprob=f)):
        with pytest.raises(ValueError):
            rq_ctx.logprobs(**dict(logits=x, token=t) | wrong)
    import recipe_dev_b200 as rq

    with pytest.raises(rq.RqError, match="0 to 64"):
        rq_ctx.logprobs(x, top_token=torch.zeros((3, 65), dtype=torch.int32, device="cuda"))
    rq_ctx.check()


@pytest.mark.parametrize("rows,vocabulary", [(1, 262144), (3, 131072), (37, 65537), (40, 262144), (148, 33000)])
@pytest.mark.parametrize("top", [1, 64])
def test_every_number_of_ctas_a_row(rq_ctx, rows, vocabulary, top):
    compare(rq_ctx, *some(rows, vocabulary, rows), top)


def test_all_alternatives_in_one_share(rq_ctx):
    """The likeliest tokens are neighbours: one CTA has them all, and few of its threads."""
    import torch

    x, token = some(5, 200001, 3)
    x[0, 150000:150064] += 50.0
    x[1, -70:] += 50.0
    x[2, :64] = torch.linspace(40.0, 41.0, 64, device="cuda")
    x[3, 77777:77787] = 60.0
    compare(rq_ctx, x, token, 64)
