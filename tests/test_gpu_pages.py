"""GPU parity of the pages of the cache (larder_amd.pages) with the oracle (oracle/pages.py): whole numbers, equal ones."""
import random

import numpy as np
import pytest
import torch

from oracle import pages as ref

pytestmark = pytest.mark.gpu


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def pool(rng, pages, n, places, page, share=0.4, fill=0.5):
    """(refs, table, lens): sequences of random lengths, some going on from another's pages, whole or not."""
    free = list(range(pages))
    rng.shuffle(free)
    free = free[:max(1, int(pages * fill))]
    table, lens = [], []
    for b in range(n):
        most = min(places, len(free))
        if b and rng.random() < share:
            other = rng.randrange(b)
            row, at = list(table[other]), rng.choice([lens[other], rng.randint(0, lens[other])])
            row = [p if i < -(-at // page) else -1 for i, p in enumerate(row)]
        else:
            at = rng.choice([0, 1, page, rng.randint(0, most * page)]) if most else 0
            row = [free.pop() for _ in range(min(most, -(-at // page)))]
            at = min(at, len(row) * page)
            row += [-1] * (places - len(row))
        table.append(row)
        lens.append(at)
    refs = [0] * pages
    for row in table:
        for p in row:
            if p >= 0:
                refs[p] += 1
    return refs, table, lens


SIZES = [(1, 1, 1, 32), (7, 3, 2, 64), (64, 5, 9, 128), (1000, 40, 30, 64), (5000, 64, 70, 32), (1024, 1500, 3, 64),
         (2048, 2100, 4, 32), (70000, 9, 1100, 64), (16384, 20, 300, 64), (16385, 3, 5, 32),
         (200000, 5, 3, 128)]


@pytest.mark.parametrize("pages,n,places,page", SIZES)
def test_take(pages, n, places, page):
    from larder_amd import pages as own
    rng = random.Random(pages + n)
    for turn in range(4):
        refs, table, lens = pool(rng, pages, n, places, page, fill=[0.5, 0.95, 1.0, 0.1][turn])
        rows = [rng.choice([0, 1, 1, 2, rng.randint(0, 3 * page)]) for _ in range(n)] if turn else [1] * n
        now = [min(x + r, places * page + 5) for x, r in zip(lens, rows)]
        cu = None if not turn else list(np.cumsum([0] + rows))
        want = ref.take(refs, table, now, cu, page)
        r, t = ints(refs), ints(table)
        got = own.take_pages(r, t, ints(now), None if cu is None else ints(cu), page=page)
        for a, b in zip((r, t, *got), want):
            assert a.tolist() == b
        # what was given is the sequences' own: a second call finds nothing to do
        if not any(want[4]):
            again = own.take_pages(r, t, ints(now), None if cu is None else ints(cu), page=page)
            assert r.tolist() == want[0] and t.tolist() == want[1]
            assert again[0].eq(-1).all() and again[1].eq(-1).all() and again[2].eq(0).all()


@pytest.mark.parametrize("pages,n,places,page", SIZES)
def test_free_and_fork(pages, n, places, page):
    from larder_amd import pages as own
    rng = random.Random(pages * 3 + n)
    refs, table, lens = pool(rng, pages, n, places, page)
    keep = [rng.choice([0, x, x + page, max(0, x - rng.randint(0, 2 * page)), -7, 2 ** 31 - 1]) for x in lens]
    want = ref.free(refs, table, keep, page)
    r, t = ints(refs), ints(table)
    own.free_pages(r, t, ints(keep), page=page)
    assert r.tolist() == want[0] and t.tolist() == want[1]
    for m in (0, 1, n, 2 * n + 3):
        parents = [rng.choice([rng.randrange(n), 0, -1, n, rng.randrange(n)]) for _ in range(m)]
        want = ref.fork(refs, table, parents)
        r, t = ints(refs), ints(table)
        new = own.fork_pages(r, t, ints(parents))
        assert r.tolist() == want[0] and new.tolist() == want[1] and t.tolist() == table
        # every place of the new table is what the pool counts
        assert sum(want[0]) == sum(p >= 0 for row in want[1] for p in row)


@pytest.mark.parametrize("pages,n,places,page", SIZES)
def test_compact(pages, n, places, page):
    from larder_amd import pages as own
    rng = random.Random(pages * 7 + n)
    refs, table, lens = pool(rng, pages, n, places, page, fill=rng.choice([0.2, 0.5, 0.9]))
    other = [[rng.choice([p, -1, pages, 2 ** 31 - 1, -2 ** 31]) for p in table[0]]]
    want = ref.compact(refs, [table, other])
    r, t, o = ints(refs), ints(table), ints(other)
    src, dst, used = own.compact_pages(r, t, o)
    m = len(want[2])
    assert r.tolist() == want[0] and t.tolist() == want[1][0] and o.tolist() == want[1][1]
    assert src.shape[0] == dst.shape[0] == max(pages // 2, 1) and used.tolist() == [want[4]]
    assert src[:m].tolist() == want[2] and dst[:m].tolist() == want[3] and src[m:].eq(-1).all() and dst[m:].eq(-1).all()


def random_cache(gen, pages, heads, width, page):
    from larder_amd import attention
    c = attention.KVCache.empty(pages, heads, width, page=page)
    for t in (c.k, c.v):
        t.view(torch.uint8).random_(0, 256, generator=gen)
    for t in (c.k_scale, c.v_scale):
        t.copy_(torch.exp2(torch.randint(-99, 99, t.shape, generator=gen, device="cuda").float()))
    return c


@pytest.mark.parametrize("heads,width,page", [(1, 64, 32), (4, 128, 64), (2, 256, 128), (3, 64, 64), (300, 64, 32)])
def test_copy(heads, width, page):
    from larder_amd import pages as own
    gen = torch.Generator(device="cuda").manual_seed(heads)
    cache = random_cache(gen, 40, heads, width, page)
    before = [t.clone() for t in cache]
    order = torch.randperm(40, generator=gen, device="cuda").int().tolist()
    src, dst = order[:15] + [-1, 40, 3, 2 ** 31 - 1, -2 ** 31], order[15:30] + [order[30], order[31], -1, order[32], order[33]]
    own.copy_pages(cache, ints(src), ints(dst))
    to = dict(zip(dst[:15], src[:15]))
    for t, old in zip(cache, before):
        raw, was = t.view(torch.uint8).flatten(1), old.view(torch.uint8).flatten(1)
        for p in range(40):
            assert torch.equal(raw[p], was[to.get(p, p)]), p


def test_offsets_that_fall_touch_nothing_else():
    """Offsets, lengths and tables of any numbers: what is outside the tensors keeps its value."""
    from larder_amd import pages as own
    rng = random.Random(5)
    for turn in range(6):
        n, places, pages = 50, 7, 33
        guard = torch.full((3, pages + 512), 77, dtype=torch.int32, device="cuda")
        refs = guard[1, 256:256 + pages]
        refs.copy_(ints([rng.choice([-5, 0, 0, 1, 2, 9]) for _ in range(pages)]))
        room = torch.full((n + 20, places), 77, dtype=torch.int32, device="cuda")
        table = room[10:10 + n]
        wild = [-2 ** 31, -1, 0, 1, 5, 31, 32, 33, 300, 2 ** 31 - 1]
        table.copy_(ints([[rng.choice(wild) for _ in range(places)] for _ in range(n)]))
        lens, cu = ints([rng.choice(wild) for _ in range(n)]), ints([rng.choice(wild) for _ in range(n + 1)])
        out = own.take_pages(refs, table, lens, cu, page=32)
        new = own.fork_pages(refs, table, ints([rng.choice(wild) for _ in range(n)]))
        own.free_pages(refs, table, lens, page=32)
        own.compact_pages(refs, table, new)
        torch.cuda.synchronize()
        assert guard[0].eq(77).all() and guard[2].eq(77).all() and guard[1, :256].eq(77).all() and guard[1, 256 + pages:].eq(77).all()
        assert room[:10].eq(77).all() and room[10 + n:].eq(77).all()
        assert all(t.shape == (n,) for t in out)


def test_steps_in_a_graph():
    """Forking, taking and copying captured once and replayed over a state that goes on, against the same steps made eagerly."""
    from larder_amd import pages as own
    rng = random.Random(11)
    pages, n, places, page = 300, 12, 6, 32
    refs, table, lens = pool(rng, pages, n, places, page, fill=0.4)
    lens = [min(x, places * page - 40) for x in lens]
    state = [ints(refs), ints(table), ints(lens)]
    gen = torch.Generator(device="cuda").manual_seed(3)
    cache = random_cache(gen, pages, 2, 64, page)
    parents = torch.zeros(n, dtype=torch.int32, device="cuda")
    got = {}

    def step(refs, table, lens, cache):
        new = own.fork_pages(refs, table, parents)
        table.copy_(new)
        lens.copy_(lens[parents.long()] + 1)
        got["out"] = own.take_pages(refs, table, lens, page=page)
        own.copy_pages(cache, got["out"][0], got["out"][1])

    mirror, held = [t.clone() for t in state], type(cache)(*[t.clone() for t in cache])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    warm, warm_cache = [t.clone() for t in state], type(cache)(*[t.clone() for t in cache])
    with torch.cuda.stream(side):
        step(*warm, warm_cache)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(*state, cache)
    out = got["out"]
    for turn in range(6):
        parents.copy_(ints([rng.randrange(n) for _ in range(n)]))
        graph.replay()
        torch.cuda.synchronize()
        step(*mirror, held)
        for a, b in zip((*state, *out), (*mirror, *got["out"])):
            assert torch.equal(a, b), turn
        for a, b in zip(cache, held):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), turn


def test_refusals():
    from larder_amd import attention, pages as own
    refs, table, i = ints([0] * 4), ints([[0, 1]] * 3), ints([1, 2, 3])
    for bad in (refs.long(), refs[None], refs[::2], refs[:0], refs.float()):
        with pytest.raises(ValueError, match="refs"):
            own.take_pages(bad, table, i)
    for bad in (table.long(), table[0], table.t(), table[:, :0]):
        with pytest.raises(ValueError, match="table"):
            own.free_pages(refs, bad, i)
    with pytest.raises(ValueError, match="lens"):
        own.take_pages(refs, table, i[:2])
    with pytest.raises(ValueError, match="cu"):
        own.take_pages(refs, table, i, i)
    with pytest.raises(ValueError, match="16 tokens"):
        own.take_pages(refs, table, i, page=16)
    with pytest.raises(ValueError, match="keep"):
        own.free_pages(refs, table, i.float())
    with pytest.raises(ValueError, match="parents"):
        own.fork_pages(refs, table, i[None])
    with pytest.raises(ValueError, match="no table"):
        own.compact_pages(refs)
    with pytest.raises(ValueError, match="devices"):
        own.free_pages(refs, table, i.cpu())
    cache = attention.KVCache.empty(4, 1, 64)
    with pytest.raises(ValueError, match="dst"):
        own.copy_pages(cache, i, i[:2])
    with pytest.raises(ValueError, match="src"):
        own.copy_pages(cache, i[None], i)
    with pytest.raises(ValueError, match="codes"):
        own.copy_pages(attention.KVCache(cache.k[::2], *cache[1:]), i, i)
