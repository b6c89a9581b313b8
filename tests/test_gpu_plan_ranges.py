"""The plan over page tables and lengths that are out of the ordinary: no slot but a true one, nothing read or written beside the arrays. GPU only (-m gpu)."""
import pytest

pytestmark = pytest.mark.gpu

MOST = 2**31 - 1


def planned(ctx, cached, fresh, table, free, page, max_tokens):
    import torch

    def dev(a):
        return torch.tensor(a, dtype=torch.int32, device="cuda")

    t = dev(table)
    got = ctx.batch_plan(dev(cached), dev(fresh), t, dev(free), page, max_tokens=max_tokens)
    ctx.check()
    return [a.tolist() for a in (t, *got)]


@pytest.mark.parametrize("entry,page", [(2**30, 16), (MOST, 16), (2**27, 16), (2**27 + 3, 16), (MOST, 2), (2**19, 4096), (2**20 + 1, 4096), (-1, 16), (-(2**31), 16)])
def test_an_entry_that_names_no_page_gives_no_slot(rq_ctx, entry, page):
    """A held page's entry from outside the cache: its positions are 2^31 or more, or below zero, and must not wrap into another page's."""
    assert not 0 <= entry * page + 1 < 2**31
    got = planned(rq_ctx, [1, 0], [1, 1], [[entry, -1], [-1, -1]], [7, 8], page, 4)
    assert got[0] == [[entry, -1], [7, -1]] and got[3] == [-1, 7 * page, -1, -1] and got[4] == [1, 0, 0, 0] and got[5] == [0, 1, -1, -1]


def test_the_last_slots_that_there_are(rq_ctx):
    """Positions just below 2^31 are slots as any others."""
    last = 2**31 // 16 - 1
    got = planned(rq_ctx, [13], [5], [[last, -1]], [last - 1], 16, 5)
    assert got[3] == [MOST - 2, MOST - 1, MOST, (last - 1) * 16, (last - 1) * 16 + 1]
    got = planned(rq_ctx, [1], [3], [[MOST, -2, -2, -2]], [5, 6, MOST], 1, 3)
    assert got[3] == [5, 6, MOST] and got[0] == [[MOST, 5, 6, MOST]]


def test_a_free_list_that_names_no_page(rq_ctx):
    got = planned(rq_ctx, [0, 0], [17, 1], [[-7, -7], [-7, -7]], [2**30, 4, -3], 16, 18)
    assert got[0] == [[2**30, 4], [-3, -7]] and got[3] == [-1] * 16 + [64, -1]


@pytest.mark.parametrize("requests", [4010, 4085, 4089, 4090, 4092, 4094, 4095, 4096])
def test_nearly_as_many_requests_as_there_can_be(requests):
    """Their lengths are just below and above what shared memory holds without being asked for; in a process of its own, where nobody has asked before."""
    import subprocess
    import sys
    from pathlib import Path

    program = f"""
import torch
import recipe_dev_b200 as rq
n = {requests}
i32 = dict(dtype=torch.int32, device="cuda")
ctx = rq.Context(0)
free = torch.arange(n, **i32).flip(0).contiguous()
got = ctx.batch_plan(torch.zeros(n, **i32), torch.ones(n, **i32), torch.full((n, 1), -1, **i32), free, 16, max_tokens=n)
ctx.check()
assert got[2].tolist() == (16 * free).tolist() and got[5].tolist() == [n, n, 0]
"""
    run = subprocess.run([sys.executable, "-c", program], capture_output=True, text=True, timeout=300, cwd=Path(__file__).resolve().parent.parent)
    assert run.returncode == 0, run.stderr[-2000:]
