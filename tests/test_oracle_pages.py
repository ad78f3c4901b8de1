"""The oracle of the pages (oracle/pages.py) against what a pool must hold, whatever is done to it: counts are the places that hold
a page, no sequence writes to a page that another holds, tokens survive forks, copies and compactions."""
import random

import pytest

from oracle import pages as ref


def counts(pages, *tables):
    refs = [0] * pages
    for t in tables:
        for row in t:
            for p in row:
                if p >= 0:
                    refs[p] += 1
    return refs


def test_take_closed_form():
    # two sequences of a page of 32: one goes on in its second page, one shares its only page with the third
    refs, table = [2, 0, 1, 0, 0], [[2, -1], [0, -1], [0, -1]]
    got = ref.take(refs, table, [33, 11, 10], [0, 1, 3, 3], 32)
    assert got == ([1, 1, 1, 1, 0], [[2, 1], [3, -1], [0, -1]], [-1, 0, -1], [-1, 3, -1], [0, 0, 0])
    # nothing is free: the place holds nothing, the share is gone
    got = ref.take([2, 1], [[0], [0], [1]], [5, 5, 5], [0, 1, 1, 1], 32)
    assert got == ([1, 1], [[-1], [0], [1]], [-1, -1, -1], [-1, -1, -1], [1, 0, 0])
    # a shared page whose tokens are all new needs no copy
    got = ref.take([2, 0], [[0], [0]], [4, 9], [0, 4, 4], 32)
    assert got == ([1, 1], [[1], [0]], [-1, -1], [-1, -1], [0, 0])


@pytest.mark.parametrize("seed", range(20))
def test_a_pool_through_many_steps(seed):
    """Tokens as (sequence of origin, place) kept beside the pages: each sequence reads its own after every operation."""
    rng = random.Random(seed)
    pages, page, places = rng.randint(20, 80), 32, 6
    n = rng.randint(1, 6)
    refs, table, lens = [0] * pages, [[-1] * places for _ in range(n)], [0] * n
    held = [[None] * page for _ in range(pages)]
    told = [[] for _ in range(n)]  # what each sequence was given
    fresh = 0
    for _ in range(60):
        what = rng.choice(["rows", "rows", "rows", "fork", "free", "compact"])
        if what == "rows":
            rows = [rng.choice([0, 1, 1, 5, 40]) for _ in lens]
            rows = [min(r, places * page - x) for r, x in zip(rows, lens)]
            now = [x + r for x, r in zip(lens, rows)]
            cu = [sum(rows[:i]) for i in range(len(rows) + 1)]
            refs, table, src, dst, lacking = ref.take(refs, table, now, cu, page)
            for a, b in zip(src, dst):
                if a >= 0:
                    held[b] = list(held[a])
            for b, (x, r) in enumerate(zip(lens, rows)):
                if lacking[b]:
                    continue
                for t in range(x, x + r):
                    p = table[b][t // page]
                    assert refs[p] == 1
                    held[p][t % page] = fresh
                    told[b].append(fresh)
                    fresh += 1
            lens = now
            # who found no page starts again
            keep = [0 if k else x for k, x in zip(lacking, lens)]
            refs, table = ref.free(refs, table, keep, page)
            told = [[] if k else t for k, t in zip(lacking, told)]
            lens = keep
        elif what == "fork":
            parents = [rng.randint(-1, len(lens) - 1) for _ in range(rng.randint(1, 6))]
            refs, table = ref.fork(refs, table, parents)
            lens, told = [lens[p] if p >= 0 else 0 for p in parents], [list(told[p]) if p >= 0 else [] for p in parents]
        elif what == "free":
            keep = [rng.choice([x, x, rng.randint(0, x)]) for x in lens]
            refs, table = ref.free(refs, table, keep, page)
            lens, told = keep, [t[:k] for t, k in zip(told, keep)]
        else:
            refs, (table,), src, dst, used = ref.compact(refs, [table])
            assert used == sum(r > 0 for r in refs) and not any(refs[used:])
            moved = [list(held[a]) for a in src]
            for b, x in zip(dst, moved):
                held[b] = x
        assert refs == counts(pages, table)
        for b, x in enumerate(lens):
            assert [held[table[b][t // page]][t % page] for t in range(x)] == told[b]
