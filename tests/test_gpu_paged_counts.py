"""assign with counts near the ends of 31 bits: its sums stop there and never wrap, so what does not fit is refused."""

import pytest
import torch

from test_gpu_paged import assign_by_hand, i32

pytestmark = pytest.mark.gpu

MOST = 2 ** 31 - 1


@pytest.fixture(scope="module")
def paged():
    from emmy_ptx import paged
    return paged


@pytest.mark.parametrize("cached, fresh, tokens", [
    ([0], [MOST], 40), ([0], [MOST - 5], 40), ([MOST], [1], 3), ([MOST - 1], [5], 9), ([MOST], [MOST], 700), ([5, MOST], [2, 0], 3), ([MOST, 7], [0, 3], 3),
    ([2, 0, 9, 1], [3, MOST, MOST, 2], 30), ([0, 2, 9, 1], [MOST, 3, 1, 2], 30), ([0, 0, 0, 0, 0], [4, 2 ** 30, 2 ** 30, 2 ** 30, 2 ** 30], 1100),
    ([0] * 1036, [1] * 1023 + [MOST] * 3 + [1] * 10, 1030), ([3] * 1030, [1] * 1022 + [MOST, 0, MOST, 0, 0, 5, 0, 1], 2000), ([0] * 2100, [2 ** 21] * 2100, 600),
    ([0] * 3000, [0] * 2999 + [MOST], 12)])
@pytest.mark.parametrize("page", [1, 16])
def test_assign_sums_that_pass_31_bits(paged, cached, fresh, tokens, page):
    width = 64 // page
    table = [[(37 * b + w) % 1000 if w * page < c else -1 for w in range(width)] for b, c in enumerate(cached)]
    free = list(range(2000, 2000 + 64 * 40))
    want_table, slots, positions, starts, lengths, head, report = assign_by_hand(cached, fresh, table, free, 0, page, tokens)
    rows = min(report[3], MOST)
    on_gpu = i32(table)
    got = paged.assign(i32(cached), i32(fresh), on_gpu, i32(free), i32([0]), page, tokens)
    assert on_gpu.tolist() == want_table
    assert got.slots.tolist() == slots and got.positions.tolist() == [min(p, MOST) for p in positions]
    assert got.starts.tolist() == [min(x, MOST) for x in starts] and got.lengths.tolist() == lengths
    assert got.free_head.tolist() == [head] and got.report.tolist() == [report[0], report[1], max(0, rows - tokens), rows]


@pytest.mark.parametrize("fresh", [2 * 10 ** 9, MOST])
def test_assign_with_table_rows_of_two_thousand_million_tokens(paged, fresh):
    """A request that its table row would hold, but not the step's rows; and one behind it."""
    table = torch.full((3, 1 << 20), -1, dtype=torch.int32, device="cuda")
    got = paged.assign(i32([0, 0, 5]), i32([7, fresh, 1]), table, i32([3, 4, 5]), i32([0]), 2047, 20)
    assert got.slots.tolist() == [3 * 2047 + i for i in range(7)] + [-1] * 13 and got.lengths.tolist() == [7, 0, 5]
    rows = min(MOST, 8 + fresh)
    assert got.starts.tolist() == [0, 7, min(MOST, 7 + fresh), rows] and got.report.tolist() == [1, 2, rows - 20, rows] and got.free_head.tolist() == [1]
    assert table[0, 0] == 3 and int((table != -1).sum()) == 1
