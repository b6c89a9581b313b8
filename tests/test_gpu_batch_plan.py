"""The plan of a serving step: page tables, slot map, positions. Whole numbers, equal to a token-by-token loop. GPU only (-m gpu)."""
import random

import pytest

from tests import serving_reference as ref

pytestmark = pytest.mark.gpu


def run(ctx, cached, fresh, table, free, page, max_tokens):
    import torch

    def dev(a):
        return torch.tensor(a, dtype=torch.int32, device="cuda")

    t = dev(table)
    got = ctx.batch_plan(dev(cached), dev(fresh), t, dev(free), page, max_tokens=max_tokens)
    return [a.tolist() for a in (t, *got)]


def a_batch(rng, n, page, most_cached, most_fresh, spare=3):
    cached, fresh = [rng.randint(0, most_cached) for _ in range(n)], [rng.randint(0, most_fresh) for _ in range(n)]
    held = [ref.pages(c, page) for c in cached]
    need = sum(ref.pages(c + f, page) - h for c, f, h in zip(cached, fresh, held))
    ids = rng.sample(range(100_000), sum(held) + need + spare)
    width = max(ref.pages(c + f, page) for c, f in zip(cached, fresh)) + 1
    table = []
    for h in held:
        table.append([ids.pop() for _ in range(h)] + [-7] * (width - h))
    return cached, fresh, table, ids


@pytest.mark.parametrize("n,page,most_cached,most_fresh", [(1, 16, 0, 1), (1, 16, 1000, 1), (3, 1, 20, 5), (64, 16, 300, 1), (255, 8, 40, 3), (256, 128, 500, 200), (257, 4096, 5000, 2), (1000, 32, 100, 70),
                                                           (4096, 16, 40, 4), (5, 16, 200, 3000)])
def test_equal_to_the_loop(rq_ctx, n, page, most_cached, most_fresh):
    rng = random.Random(n * page)
    batch = a_batch(rng, n, page, most_cached, most_fresh)
    total = sum(batch[1])
    for max_tokens in (total + 17, max(1, total - 1)):  # padding behind the batch, and arrays that are too short for it
        assert run(rq_ctx, *batch, page, max_tokens) == list(map(list, ref.plan(*batch, page, max_tokens)))
    rq_ctx.check()


def test_requests_without_new_tokens_and_lengths_at_page_ends(rq_ctx):
    cached, fresh = [0, 16, 15, 32, 16, 0, 0], [0, 0, 1, 1, 17, 16, 0]
    table = [[-1] * 4, [3, -1, -1, -1], [4, -1, -1, -1], [5, 6, -1, -1], [7, -1, -1, -1], [-1] * 4, [-1] * 4]
    free = [20, 21, 22, 23, 24]
    got = run(rq_ctx, cached, fresh, table, free, 16, 40)
    assert got == list(map(list, ref.plan(cached, fresh, table, free, 16, 40)))
    assert got[6] == [35, 4, 0]  # tokens, pages taken, none lacking


def test_a_list_that_is_too_short_and_a_table_that_is_too_narrow(rq_ctx):
    cached, fresh = [10, 0, 30, 5], [10, 40, 40, 1]
    table = [[0, -1, -1], [-1, -1, -1], [1, 2, -1], [3, -1, -1]]
    for free in ([50, 51, 52], [50], []):
        got = run(rq_ctx, cached, fresh, table, free, 16, 100)
        assert got == list(map(list, ref.plan(cached, fresh, table, free, 16, 100))), free
        assert got[6][2] > 0


def test_negative_lengths_count_as_zero_and_planning_again_changes_nothing(rq_ctx):
    import torch

    cached, fresh, free = [5, -3, 20], [1, 2, -9], [9, 8, 7]
    table = [[1, -1], [-1, -1], [2, 3]]
    want = list(map(list, ref.plan(cached, fresh, table, free, 16, 8)))
    assert run(rq_ctx, cached, fresh, table, free, 16, 8) == want
    dev = [torch.tensor(a, dtype=torch.int32, device="cuda") for a in (cached, fresh, table, free)]
    for _ in range(2):
        got = rq_ctx.batch_plan(*dev, 16, max_tokens=8)
    assert [a.tolist() for a in (dev[2], *got)] == want


def test_refusals(rq_ctx):
    import torch

    import recipe_dev_b200 as rq

    i = torch.zeros(8, dtype=torch.int32, device="cuda")
    table = torch.zeros((2, 4), dtype=torch.int32, device="cuda")
    for page in (0, 3, 8192, -16):
        with pytest.raises(rq.RqError, match="power of two"):
            rq_ctx.batch_plan(i[:2], i[:2], table, i, page, max_tokens=4)
    with pytest.raises(ValueError):
        rq_ctx.batch_plan(i[:2], i[:2], table, i, 16)  # no size for the per-token arrays
    with pytest.raises(ValueError):
        rq_ctx.batch_plan(i[:2].float(), i[:2], table, i, 16, max_tokens=4)
    with pytest.raises(ValueError):
        rq_ctx.batch_plan(i[:3], i[:3], table, i, 16, max_tokens=4)  # fewer rows in the table than requests
    many = torch.zeros(4097, dtype=torch.int32, device="cuda")
    with pytest.raises(rq.RqError, match="4096"):
        rq_ctx.batch_plan(many, many, torch.zeros((4097, 1), dtype=torch.int32, device="cuda"), i, 16, max_tokens=4)
    a = [i.data_ptr()] * 2
    assert rq_ctx.lib.rq_batch_plan(rq_ctx.handle, *a, 2, 16, table.data_ptr(), 3, 4, i.data_ptr(), 8, *[i.data_ptr()] * 5, 4, i.data_ptr(), None) == -1  # rows that overlap
    assert rq_ctx.lib.rq_batch_plan(rq_ctx.handle, *a, 2, 16, None, 4, 4, i.data_ptr(), 8, *[i.data_ptr()] * 5, 4, i.data_ptr(), None) == -1
    rq_ctx.check()
