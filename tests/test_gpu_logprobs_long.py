"""Log probabilities of rows that a CTA has many rounds of, several a segment, and of more rows than the GPU has clusters for. GPU only (-m gpu).

Bounds: test_gpu_logprobs.py's, which hold a thread's chain of up to 64 rounds; where one CTA takes more, its chain is longer by the rounds beyond, and so is the bound on a sum."""
import pytest

from tests.test_gpu_logprobs import compare, run, some

pytestmark = pytest.mark.gpu


class Held:
    """Gives a few rows of one call's outputs to what compares them."""

    def __init__(self, out, rows):
        self.out, self.rows = out, rows

    def logprobs(self, logits, token, **given):
        for name, a in given.items():
            a.copy_(self.out[name][self.rows])
        return given["logprob"]

    def check(self):
        pass


def compare_in_parts(ctx, x, token, top, step=20):
    out = run(ctx, x, token, top)
    for r in range(0, x.shape[0], step):
        rows = slice(r, r + step)
        compare(Held(out, rows), x[rows], token[rows], top)


def ordered(x, order):
    import torch

    if order == "rising":
        return torch.sort(x, dim=1).values.contiguous()
    if order == "equal":
        return torch.full_like(x, -3.25)
    if order == "two sizes":
        return torch.where(x > 0, 1.0, 0.0)
    if order == "one share":  # all alternatives are neighbours, of one thread's rounds and the next one's
        x[:, -3000:-2900] += 60.0
    return x


# A CTA a row, of 64 rounds (four a segment), 18 and 17 (two; the ninth segment whole, and half empty); two CTAs of 37 rounds (three), eight of 31
@pytest.mark.parametrize("rows,vocabulary", [(300, 262144), (297, 70001), (299, 66000), (150, 300007), (40, 1000003)])
@pytest.mark.parametrize("top", [20, 64])
@pytest.mark.parametrize("order", ["random", "rising", "equal", "two sizes", "one share"])
def test_many_rounds_a_segment(rq_ctx, rows, vocabulary, top, order):
    x, token = some(rows, vocabulary, rows)
    x = ordered(x, order)
    compare_in_parts(rq_ctx, x, token, top)


@pytest.mark.parametrize("rows,vocabulary", [(2039, 32000), (700, 40001)])
@pytest.mark.parametrize("order", ["random", "equal", "rising"])
def test_prompts_with_alternatives(rq_ctx, rows, vocabulary, order):
    """A CTA a row, whose own part of the list overflows where logits are equal, in all rows at once."""
    x, token = some(rows, vocabulary, rows)
    x = ordered(x, order)
    compare_in_parts(rq_ctx, x, token, 20, step=200)


def test_masked_rows_of_many_rounds(rq_ctx):
    import torch

    x, token = some(300, 70001, 5, offset=1, pad=2)
    x[0, ::2], x[1, 1::2], x[2, 60000:], x[3, :60000], x[4] = -torch.inf, float("nan"), -torch.inf, float("nan"), torch.finfo(torch.float32).min
    x[5, 50:] = -torch.inf
    token[:8] = torch.tensor([2, 3, 69999, 5, 70000, 49, -1, 70001], dtype=torch.int32)
    compare_in_parts(rq_ctx, x, token, 64)


def test_more_than_2_to_the_31_logits(rq_ctx):
    import torch

    rows, vocabulary = 8300, 262144
    x = torch.empty((rows, vocabulary), device="cuda")
    assert x.numel() > 2**31
    gen = torch.Generator(device="cuda").manual_seed(0)
    for r in range(0, rows, 830):
        x[r : r + 830].normal_(0.0, 2.5, generator=gen)
    token = torch.randint(0, vocabulary, (rows,), generator=gen, device="cuda").int()
    out = run(rq_ctx, x, token, 20)
    for part in (slice(0, 3), slice(8190, 8194), slice(rows - 3, rows)):
        compare(Held(out, part), x[part], token[part], 20)
    assert (out["rank"] >= 0).all() and (out["logprob"] < 0).all()
