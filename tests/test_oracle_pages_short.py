"""The oracle of the pages where a pool has run out: a page that several sequences share is lost to none as long as one can keep it."""
import random

import pytest

from oracle import pages as ref


def test_the_last_holder_keeps_its_page():
    # two holders, nothing free: the second goes on in the page
    assert ref.take([2, 1, 1], [[0, -1], [0, -1]], [5, 5], None, 32) == ([1, 1, 1], [[-1, -1], [0, -1]], [-1, -1], [-1, -1], [1, 0])
    # one page free: the first has it and copies, the second goes on
    assert ref.take([2, 0], [[0], [0]], [5, 5], None, 32) == ([1, 1], [[1], [0]], [0, -1], [1, -1], [0, 0])
    # enough pages: both copy, as ever
    assert ref.take([2, 0, 0], [[0], [0]], [5, 5], None, 32) == ([0, 1, 1], [[1], [2]], [0, 0], [1, 2], [0, 0])
    # three holders, of whom one writes nothing: it alone holds the page then
    assert ref.take([3, 1], [[0], [0], [0]], [5, 5, 5], [0, 1, 1, 2], 32) == ([1, 1], [[-1], [0], [-1]], [-1] * 3, [-1] * 3, [1, 0, 1])
    # all three write
    assert ref.take([3, 1], [[0], [0], [0]], [5, 5, 5], None, 32) == ([1, 1], [[-1], [-1], [0]], [-1] * 3, [-1] * 3, [1, 1, 0])


@pytest.mark.parametrize("seed", range(30))
def test_no_shared_page_is_lost(seed):
    """Pools of few free pages: counts are the places, what a sequence keeps is its own, and every page that was held is held still
    or was copied for each of its holders."""
    rng = random.Random(seed)
    n, groups = rng.randint(2, 9), rng.randint(1, 4)
    pages = groups + rng.randint(0, 3)
    table = [[rng.randrange(groups), -1] for _ in range(n)]
    refs = [sum(row[0] == p for row in table) for p in range(pages)]
    rows = [rng.choice([0, 1, 1, 1, 30]) for _ in range(n)]
    lens = [5 + r for r in rows]
    got, new, src, dst, lacking = ref.take(refs, table, lens, [sum(rows[:i]) for i in range(n + 1)], 32)
    assert got == [sum(p == q for row in new for q in row) for p in range(pages)]
    for b in range(n):
        if rows[b] and new[b][0] >= 0:
            assert got[new[b][0]] == 1
    for p in range(groups):
        holders = [b for b in range(n) if table[b][0] == p]
        if holders and not got[p]:
            assert all(src[b] == p and dst[b] == new[b][0] >= 0 for b in holders)
