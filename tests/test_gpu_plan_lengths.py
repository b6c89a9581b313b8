"""The plan over lengths whose sum passes what 32 bits hold: sums end at 2^31 - 1, tokens past the table's width have no slot, and the others of the batch are
planned as ever. GPU only (-m gpu)."""
import pytest

from tests.test_gpu_plan_ranges import MOST, planned

pytestmark = pytest.mark.gpu


def expected(cached, fresh, table, free, page, max_tokens):
    table = [list(row) for row in table]
    width, taken, lacking, total = len(table[0]), 0, 0, 0
    starts, slots, positions, owners = [0], [], [], []
    for r, (c, f) in enumerate(zip(cached, fresh)):
        held, every = -(-c // page), -(-(c + f) // page)
        columns = range(held, max(held, min(every, width)))
        lacking += every - held - len(columns)
        for column in columns:
            table[r][column] = free[taken] if taken < len(free) else -1
            lacking += taken >= len(free)
            taken += taken < len(free)
        for position in range(c, c + min(f, max_tokens - len(slots))):
            entry = table[r][position // page] if position // page < width and position <= MOST else -1
            slots.append(entry * page + position % page if entry >= 0 else -1)
            positions.append(min(position, MOST))
            owners.append(r)
        total += f
        starts.append(min(total, MOST))
    pad = max_tokens - len(slots)
    status = [starts[-1], taken, min(lacking, MOST)]
    return [table, starts, [min(c + f, MOST) for c, f in zip(cached, fresh)], slots + [-1] * pad, positions + [0] * pad, owners + [-1] * pad, status]


@pytest.mark.parametrize("page", [1, 16, 4096])
@pytest.mark.parametrize("cached,fresh", [(MOST, 3), (MOST - 1, 3), (MOST - 15, 20), (MOST - 16, 20), (2**30, 3), (MOST, MOST), (5, MOST), (MOST, 0), (0, MOST)])
def test_lengths_past_the_table(rq_ctx, cached, fresh, page):
    batch = [2, cached, 4], [1, fresh, 2], [[30, 29, -1], [31, 32, 28], [33, 34, 35]], [7, 8, 9, 10], page, 9
    assert planned(rq_ctx, *batch) == expected(*batch)


def test_many_requests_of_more_tokens_than_32_bits_count(rq_ctx):
    n = 300
    batch = [0] * n, [2**24] * n, [[-1]] * n, list(range(n)), 16, 40
    got = planned(rq_ctx, *batch)
    assert got == expected(*batch) and got[6] == [MOST, n, n * (2**20 - 1)]
    batch = [0] * 4096, [MOST] * 4096, [[-1]] * 4096, [9], 1, 3
    got = planned(rq_ctx, *batch)
    assert got == expected(*batch) and got[6] == [MOST, 1, MOST]
