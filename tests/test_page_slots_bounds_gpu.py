"""page_slots at the end of what positions, slots and tables can be: numbers that 32 bits do not hold are given no slot."""
import pytest
import torch

import miori_b200 as mb

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
MOST = 2 ** 31 - 1


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def plain(held, new, table, pool, page, T):
    """Token by token in whole numbers without end."""
    width, given, slots, positions = len(table[0]), 0, [], []
    for r, (h, n) in enumerate(zip(held, new)):
        after = min(h + n, MOST)
        for i in range(min(-(-h // page), width), min(-(-after // page), width)):
            table[r][i] = pool[given] if given < len(pool) else -1
            given += 1
        for p in range(h, h + n):
            number = table[r][p // page] if p // page < width and p < MOST else -1
            slot = number * page + p % page if number >= 0 else -1
            slots.append(slot if slot <= MOST else -1)
            positions.append(min(p, MOST))
    return (slots + [-1] * T)[:T], (positions + [0] * T)[:T], [min(h + n, MOST) for h, n in zip(held, new)], given


@pytest.mark.parametrize("held,new,page,width", [
    ([MOST - 10, 5], [20, 3], 1 << 20, 2048),       # past the last position
    ([MOST, MOST - 1, 0], [3, 2, 1], 1 << 24, 130),
    ([MOST - 40], [45], 1 << 30, 2),
    ([MOST - 40, MOST], [45, 1], 1 << 30, 1),         # and past the table
    ([0, 7], [30, 4], 1 << 30, 3),
    ([(1 << 30) - 2], [4], 1 << 30, 2)])
def test_positions_and_slots_that_int32_does_not_hold(held, new, page, width):
    numbers = [0, 1, 5, 2047, 2048, 4000, MOST]  # of pages: whose slots int32 holds, or not
    table = [[numbers[(3 * r + c) % 7] if c < min(-(-h // page), width) else -1 for c in range(width)] for r, h in enumerate(held)]
    pool, T = [6, 1, 2 ** 30, 0, MOST], sum(new) + 2
    t = i32(table)
    got = mb.page_slots(i32(held), i32(new), t, i32(pool), i32([0]), page, T)
    torch.cuda.synchronize()
    slots, positions, after, given = plain(held, new, table, pool, page, T)
    assert got[0].tolist() == slots and got[1].tolist() == positions and got[3].tolist() == after and int(got[4]) == given
    assert t.tolist() == table


def test_refusals():
    a, one = i32([1, 2]), i32([0])
    with pytest.raises(mb.MioriError, match="2.30 positions"):
        mb.page_slots(a, a, torch.zeros(2, 4, dtype=torch.int32, device=DEV), a, one, 2 ** 30 + 1, 4)
