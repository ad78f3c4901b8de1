"""GPU parity of the attention of chunks of rows over the paged cache (larder_amd.attention.chunk_rows) against the float64 oracle
(oracle/attention.py), and a run of norms, pages, appending and chunks together.

Tolerances: attention_bound of test_gpu_attention.py, whose terms are what the kernels round, with weights rounded to q's type."""
import random

import numpy as np
import pytest
import torch

from oracle import attention as ref
from oracle import pages as pool_ref
from test_gpu_attention import (BF16, F16, attention_bound, cache_host, cu_of, host, ints, normal, page_table,  # noqa: F401
                                poisoned_memory, random_cache)

pytestmark = pytest.mark.gpu


def check(got, q, cache, table, lens, cu, scale, dtype, over=4.0):
    """Every row against the oracle (several hundred rows and keys at most)."""
    codes = cache_host(cache)
    qh = host(q)
    for b, n in enumerate(lens):
        if cu[b + 1] == cu[b]:
            continue
        x = qh[cu[b]:cu[b + 1]]
        k, there = ref.read(*codes[0], table[b], n)
        v, _ = ref.read(*codes[1], table[b], n)
        want, spread = ref.attend(x, k, v, scale, there)
        have = host(got[cu[b]:cu[b + 1]])
        bound = attention_bound(x, k, scale, want, spread, dtype, dtype)
        assert np.array_equal(np.isnan(have), np.isnan(want)), b
        ok = (np.abs(have - want) <= bound) | np.isnan(want)
        assert ok.all(), (b, n, np.abs(have - want)[~ok].max(), bound[~ok].min())


def check_long(got, q, cache, table, lens, cu, scale, dtype, some=None):
    """The same against float64 on the GPU, whole heads at a time; finite caches without holes."""
    page = cache.k.shape[2]
    hq, hk, width = q.shape[1], cache.k.shape[1], q.shape[2]
    g = hq // hk
    for b, n in enumerate(lens):
        r = cu[b + 1] - cu[b]
        if r == 0:
            continue
        pages = torch.as_tensor(table[b, :-(-n // page)].astype(np.int64)).cuda()
        k, v = ((c[pages].double() * s[pages].double()[..., None, None]).transpose(0, 1).flatten(1, 2)[:, :n]
                for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
        seen = torch.arange(n, device="cuda") <= torch.arange(n - r, n, device="cuda")[:, None]
        for h in (range(hq) if some is None else some):
            x = q[cu[b]:cu[b + 1], h].double()
            kh, vh = k[h // g].contiguous(), v[h // g].contiguous()
            p = torch.softmax((x @ kh.t() * scale).masked_fill(~seen, float("-inf")), -1).nan_to_num(0.0)
            want, spread = p @ vh, p @ vh.abs()
            top = (x.abs() @ kh.abs().t()).amax(-1, keepdim=True) * scale
            weight = torch.finfo(dtype).eps / 2 + (width + 8) * 2.0 ** -24 * top + 2.0 ** -19
            bound = torch.finfo(dtype).eps / 2 * want.abs() + 2 * weight * spread + (2.0 ** -25 if dtype == F16 else 0) + 1e-30
            off = (got[cu[b]:cu[b + 1], h].double() - want).abs()
            assert (off <= bound).all(), (b, h, (off - bound).max().item())


HEADS = [(4, 4, 64, 32), (8, 1, 128, 64), (7, 1, 128, 32), (16, 2, 256, 64), (40, 2, 64, 128), (3, 3, 256, 128), (12, 4, 128, 128),
         (200, 1, 64, 32), (2, 2, 128, 32), (9, 1, 256, 32)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("q_heads,heads,width,page", HEADS)
@pytest.mark.parametrize("longest", [None, 64])
def test_chunk(dtype, q_heads, heads, width, page, longest):
    """Chunks and lengths of 0, 1, a tile's and a page's ends and odd ones; more rows than tokens; rows of no sequence."""
    from larder_amd import attention
    rng = np.random.default_rng(q_heads + width)
    rows = [0, 1, 17, 3, 40, 2, 33, 16, 5]
    lens = [40, 1, 17, 2, 300, page, page + 33, 3 * page + 1, 0]
    cu = [3] + [3 + x for x in np.cumsum(rows)]
    table, n = page_table(rng, [-(-x // page) for x in lens], width=12)
    cache = random_cache(rng, n, heads, width, page)
    q = normal(rng, cu[-1] + 4, q_heads, width, dtype=dtype)
    got = attention.chunk_rows(q, cache, ints(table), ints(lens), ints(cu), longest=longest)
    assert (got[:3] == 0).all() and (got[cu[-1]:] == 0).all() and (got[cu[3]:cu[3] + 1] == 0).all() and (got[cu[8]:cu[9]] == 0).all()
    check(got, q, cache, table, lens, cu, width ** -0.5, dtype)
    # another scale, views of a wider product
    wide = normal(rng, cu[-1] + 4, q_heads + 3, width, dtype=dtype)
    got = attention.chunk_rows(wide[:, 2:2 + q_heads], cache, ints(table), ints(lens), ints(cu), longest=longest, scale=0.3)
    check(got, wide[:, 2:2 + q_heads], cache, table, lens, cu, 0.3, dtype)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("q_heads,heads,width,page,rows,lens", [
    (4, 4, 64, 32, [700], [700]), (8, 1, 128, 64, [129, 500], [5000, 500]), (28, 4, 128, 32, [64, 200, 31], [4097, 1000, 9000]),
    (4, 2, 256, 64, [300], [4500]), (6, 2, 256, 128, [1, 90], [4200, 8300]), (1, 1, 128, 128, [1500], [1500]),
    (16, 2, 64, 64, [40] * 9, [4100, 64, 40, 1000, 41, 129, 8191, 8192, 8193]), (32, 4, 128, 64, [48], [20000]),
    (4, 1, 64, 32, [2000], [6000]), (32, 4, 128, 64, [2048], [4096]), (32, 4, 128, 32, [600], [9001]), (16, 2, 128, 128, [5], [40000])])
@pytest.mark.parametrize("longest", [None, 100])
def test_chunk_long(dtype, q_heads, heads, width, page, rows, lens, longest):
    """Past 64 tiles of keys; keys in chunks (longest None) and in one (100)."""
    from larder_amd import attention
    rng = np.random.default_rng(sum(lens))
    cu = cu_of(rows)
    table, n = page_table(rng, [-(-x // page) for x in lens])
    cache = random_cache(rng, n, heads, width, page)
    q = normal(rng, cu[-1], q_heads, width, dtype=dtype, scale=2.0)
    got = attention.chunk_rows(q, cache, ints(table), ints(lens), ints(cu), longest=longest)
    check_long(got, q, cache, table, lens, cu, width ** -0.5, dtype, some=sorted({0, q_heads // 2, q_heads - 1}))
    again = attention.chunk_rows(q, cache, ints(table), ints(lens), ints(cu), longest=longest)
    assert torch.equal(got, again)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n,rows", [(65, 1), (300, 1), (70, 9), (200, 33)])
def test_chunk_many_sequences(dtype, n, rows):
    """More sequences than a wavefront has lanes: one row each without offsets, and ragged ones, empty ones among them."""
    from larder_amd import attention
    rng = np.random.default_rng(n)
    lens = [int(x) for x in rng.choice([0, 1, 31, 64, 65, 200], n)]
    table, pages = page_table(rng, [-(-x // 32) for x in lens], width=7)
    cache = random_cache(rng, pages, 2, 64, 32)
    if rows == 1:
        q, cu = normal(rng, n, 6, 64, dtype=dtype), list(range(n + 1))
        got = attention.chunk_rows(q, cache, ints(table), ints(lens))
    else:
        counts = [int(x) for x in rng.choice([0, 1, rows, 2 * rows], n)]
        cu = cu_of(counts)
        q = normal(rng, cu[-1] + 2, 6, 64, dtype=dtype)
        got = attention.chunk_rows(q, cache, ints(table), ints(lens), ints(cu))
        assert (got[cu[-1]:] == 0).all()
    check(got, q, cache, table, lens, cu, 0.125, dtype)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("q_heads,heads,width,page", [(7, 1, 128, 32), (4, 4, 64, 32), (16, 1, 256, 64), (3, 3, 128, 128), (200, 1, 64, 32)])
@pytest.mark.parametrize("kind", ["few", "many", "one"])
def test_chunk_far_shorter_than_said(dtype, q_heads, heads, width, page, kind):
    """`longest` far above the lengths, so that a call is laid out for long ones: few and short pieces, tiles that are shared and
    tiles that are not, sequences without rows between, more than 64 of them in a row, rows before and behind."""
    from larder_amd import attention
    rng = np.random.default_rng(31 * q_heads + width)
    if kind == "few":
        rows, lens = [5, 0, 90, 1, 0, 33], [200, 64, 1500, 129, 3, 1021]
    elif kind == "one":
        rows, lens = [130], [777]
    else:
        rows = [int(x) for x in rng.choice([0, 1, 2, 40], 90)] + [0] * 150 + [3] + [0] * 70 + [65, 0]
        lens = [int(x) for x in rng.choice([0, 1, 63, 65, 300, 500], len(rows))]
    cu = [2] + [2 + int(x) for x in np.cumsum(rows)]
    table, n = page_table(rng, [-(-x // page) for x in lens], width=65536 // page)
    cache = random_cache(rng, n, heads, width, page)
    q = normal(rng, cu[-1] + 3, q_heads, width, dtype=dtype)
    got = attention.chunk_rows(q, cache, ints(table), ints(lens), ints(cu))
    assert (got[:2] == 0).all() and (got[cu[-1]:] == 0).all()
    check(got, q, cache, table, lens, cu, width ** -0.5, dtype)
    assert torch.equal(got, attention.chunk_rows(q, cache, ints(table), ints(lens), ints(cu)))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("longest", [None, 64])
@pytest.mark.parametrize("page,heads,width", [(32, 2, 128), (64, 1, 64), (32, 1, 256)])
def test_chunk_holes_and_nan(dtype, longest, page, heads, width):
    """Pages that are not there are not seen; NaN behind the last token or in pages of others is not met, NaN in a seen key or
    value reaches the rows that see it and no other."""
    from larder_amd import attention
    rng = np.random.default_rng(12)
    rows, lens = [40, 4, 70, 1], [page * 3 + 4, page * 2 + 6, page * 2 + 26, 40]
    cu = cu_of(rows)
    table, n = page_table(rng, [4, 3, 3, 2], width=5)
    table[0, 1], table[2, 0] = -1, 2 ** 31 - 1
    cache = random_cache(rng, n, heads, width, page)
    k, v = cache.k.view(torch.uint8), cache.v.view(torch.uint8)
    for b, m in enumerate(lens):  # behind the last token
        if 0 <= table[b, m // page] < n:
            k[int(table[b, m // page]), :, m % page:] = 0x7f
            v[int(table[b, m // page]), :, m % page:] = 0xff
    v[int(table[1, 2]), 0, 5, 5] = 0x7f          # the last token of sequence 1: its last row alone
    v[int(table[1, 2]), heads - 1, 4, 7] = 0xff  # the one before: the last two
    k[int(table[2, 2]), 0, 20, 9] = 0x7f         # a key that the last rows of sequence 2 see
    v[int(table[2, 1]), 0, 3, width - 1] = 0x7f  # a value that many of its rows see, and some do not
    q = normal(rng, cu[-1], 4 * heads, width, dtype=dtype)
    got = attention.chunk_rows(q, cache, ints(table), ints(lens), ints(cu), longest=longest)
    check(got, q, cache, table, lens, cu, width ** -0.5, dtype)
    assert torch.isnan(got[43, :4, 5]).all() and not torch.isnan(got[42, :4, 5]).any()
    # a page that is not there, far before the rows, in a cache whose first page is all NaN
    far, most = page_table(rng, [9], width=9)
    far = far + 1
    deep = random_cache(rng, most + 1, heads, width, page)
    for t in (deep.k, deep.v):
        t.view(torch.uint8)[0] = 0x7f
    far[0, 2] = -1
    few = q[:40]
    got = attention.chunk_rows(few, deep, ints(far), ints([9 * page]), ints([0, 40]), longest=longest)
    check(got, few, deep, far, [9 * page], [0, 40], width ** -0.5, dtype)
    assert not torch.isnan(got).any()
    # a sequence none of whose pages is there, whatever the first page of the cache holds
    v[0], k[0] = 0x7f, 0x7f
    gone = attention.chunk_rows(q, cache, ints(np.full_like(table, n)), ints(lens), ints(cu), longest=longest)
    assert (gone == 0).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("page", [32, 64])
def test_chunk_scales_of_all_sizes(dtype, page):
    """Pages whose scales of keys and values lie far apart: a row's own pages decide what it gives (float16: values from 2^-24
    to 2^15, pages beside each other within 2^22)."""
    from larder_amd import attention
    rng = np.random.default_rng(5)
    lens, rows = [page * 9 + 5, 200], [60, 130]
    cu = cu_of(rows)
    table, n = page_table(rng, [-(-x // page) for x in lens], width=10)
    cache = random_cache(rng, n, 1, 64, page)
    steps = [-24, -12, 6, -9, -20, 0, -5, 5, -16, -2] if dtype == F16 else [-90, 60, -30, 100, 0, -60, 3, -100, 90, -8]
    for b in range(2):
        for i in range(-(-lens[b] // page)):
            p = int(table[b, i])
            cache.v_scale[p] = 2.0 ** steps[(i + 3 * b) % 10]
            cache.k_scale[p] = 2.0 ** (-8 + (i % 3))
    q = normal(rng, cu[-1], 3, 64, dtype=dtype)
    q[::5] = 0  # rows that see all of their tokens alike
    for longest in (None, 64):
        got = attention.chunk_rows(q, cache, ints(table), ints(lens), ints(cu), longest=longest)
        check(got, q, cache, table, lens, cu, 0.125, dtype)


def test_chunk_scores_of_minus_infinity_and_large_ones():
    """Scores past float32 are infinite: rows whose every score is -infinity attend to nothing; large finite ones pick one token."""
    from larder_amd import attention
    cache = attention.KVCache.empty(4, 1, 64, 64)
    cache.k.view(torch.uint8).fill_(0x38)  # ones
    cache.v.view(torch.uint8).fill_(0x40)  # twos
    cache.k_scale.fill_(2.0 ** 20), cache.v_scale.fill_(1.0)
    table, lens, cu = ints([[2, 0, 3]]), ints([150]), ints([0, 40])
    q = torch.full((40, 2, 64), 1.0, dtype=BF16, device="cuda")
    q[:20] = -3e38
    got = attention.chunk_rows(q, cache, table, lens, cu)
    assert (got[:20] == 0).all() and (got[20:] == 2).all()
    rng = np.random.default_rng(8)
    cache = random_cache(rng, 4, 1, 64, 64)
    q = normal(rng, 40, 2, 64, dtype=BF16, scale=200.0)
    check(attention.chunk_rows(q, cache, table, lens, cu), q, cache, np.array([[2, 0, 3]]), [150], [0, 40], 0.125, BF16)


def test_chunk_keeps_small_weights():
    """A token that stands out over 8,191 that weigh 2^-20 of it each: together 2^-7."""
    from larder_amd import attention
    page, n = 64, 128
    cache = attention.KVCache.empty(n, 1, 64, page)
    k, v = torch.zeros(n, 1, page, 64), torch.zeros(n, 1, page, 64)
    k[0, 0, 0, 0], v[..., 1] = 16.0, 1.0
    v[0, 0, 0, 1] = 0.0
    for codes, x in ((cache.k, k), (cache.v, v)):
        codes.view(torch.uint8).copy_(x.to(torch.float8_e4m3fn).view(torch.uint8))
    cache.k_scale.fill_(1.0), cache.v_scale.fill_(1.0)
    table, lens, cu = torch.arange(n, dtype=torch.int32, device="cuda")[None], ints([n * page]), ints([0, 20])
    for dtype in (F16, BF16):
        q = torch.zeros(20, 1, 64, dtype=dtype, device="cuda")
        q[:, 0, 0] = 0.8672  # 20.02 octaves at scale 1
        for longest in (None, 128):
            got = attention.chunk_rows(q, cache, table, lens, cu, longest=longest, scale=1.0)
            w = (n * page - 1) * np.exp(-16.0 * float(q[19, 0, 0]))
            want = w / (1 + w)
            assert abs(float(got[19, 0, 1]) / want - 1) <= 3 * torch.finfo(dtype).eps / 2 + 2.0 ** -19


def test_chunk_offsets_past_32_bits():
    """Pages past 2^32 bytes of codes."""
    from larder_amd import attention
    pages = 2 ** 32 // (8 * 128 * 256) + 40
    cache = attention.KVCache.empty(pages, 8, 256, 128)
    rng = np.random.default_rng(3)
    near = random_cache(rng, 6, 8, 256, 128)
    table = np.array([[pages - 1, 3, pages - 20, 1], [pages - 7, pages - 2, 0, 0]])
    for i, p in enumerate([pages - 1, 3, pages - 20, 1, pages - 7, pages - 2]):
        for a, c in zip(cache, near):
            a[p].view(torch.uint8).copy_(c[i].view(torch.uint8))
    q = normal(rng, 50, 8, 256, dtype=F16)
    lens, cu = [450, 200], [0, 20, 50]
    got = attention.chunk_rows(q, cache, ints(table), ints(lens), ints(cu))
    small = np.array([[0, 1, 2, 3], [4, 5, 0, 0]])
    assert torch.equal(got, attention.chunk_rows(q, near, ints(small), ints(lens), ints(cu), longest=512))
    check_long(got, q, near, small, lens, cu, 1 / 16, F16)


def test_chunk_wrong_numbers_touch_nothing_else():
    """Offsets, lengths and tables of any numbers: rows have no meaning then, and the rows around the output keep their values."""
    from larder_amd import attention
    rng = np.random.default_rng(4)
    cache = random_cache(rng, 9, 1, 64, 32)
    wild = [-2 ** 31, -5, -1, 0, 1, 7, 30, 64, 100, 2 ** 31 - 1]
    for n in (1, 5, 64, 65, 200):
        for turn in range(3):
            pick = random.Random(n * 10 + turn)
            q = normal(rng, 100, 3, 64, dtype=BF16)
            cu = ints([pick.choice(wild) for _ in range(n + 1)])
            lens = ints([pick.choice(wild) for _ in range(n)])
            table = ints([[pick.choice(wild) for _ in range(4)] for _ in range(n)])
            kept = [t.clone() for t in cache]
            print("wild", n, turn, flush=True)
            attention.chunk_rows(q, cache, table, lens, cu, longest=pick.choice([None, 1, 128]))
            torch.cuda.synchronize()
            assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(cache, kept))


def test_chunk_and_single_rows_agree():
    """attend_rows and chunk_rows are one sum in two orders."""
    from larder_amd import attention
    rng = np.random.default_rng(9)
    lens, rows = [1000, 77, 500], [20, 77, 1]
    cu = cu_of(rows)
    table, n = page_table(rng, [-(-x // 64) for x in lens])
    cache = random_cache(rng, n, 2, 128, 64)
    q = normal(rng, cu[-1], 16, 128, dtype=F16)
    a = attention.attend_rows(q, cache, ints(table), ints(lens), cu=ints(cu))
    b = attention.chunk_rows(q, cache, ints(table), ints(lens), ints(cu))
    assert (a.float() - b.float()).abs().max() <= 4 * 2.0 ** -11 * a.float().abs().max()


def test_chunk_in_a_graph_and_on_streams():
    from larder_amd import attention
    rng = np.random.default_rng(6)
    lens, rows = [3000, 400], [60, 30]
    cu = cu_of(rows)
    table, n = page_table(rng, [-(-x // 64) for x in lens])
    cache = random_cache(rng, n, 2, 128, 64)
    q, tab, ln, off = normal(rng, 90, 8, 128), ints(table), ints(lens), ints(cu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = attention.chunk_rows(q, cache, tab, ln, off)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, attention.chunk_rows(q, cache, tab, ln, off))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = attention.chunk_rows(q, cache, tab, ln, off)
    for turn in range(4):
        q.copy_(normal(rng, 90, 8, 128))
        ln.copy_(ints([3000 - 700 * turn, 400 - 99 * turn]))
        graph.replay()
        torch.cuda.synchronize()
        eager = attention.chunk_rows(q, cache, tab, ln, off)
        assert torch.equal(out, eager), turn
    check_long(out, q, cache, table, [900, 103], cu, 128 ** -0.5, BF16)


def test_chunk_refusals():
    from larder_amd import attention
    cache = attention.KVCache.empty(4, 2, 64)
    q, table, lens, cu = torch.zeros(6, 4, 64, dtype=F16, device="cuda"), ints([[0, 1]]), ints([9]), ints([0, 6])
    for kw, why in ((dict(q=q.float()), "float16 or bfloat16"), (dict(q=q[:, :3]), "3 query heads"), (dict(q=q[..., :32]), "q is"),
                    (dict(cu=None), "offsets"), (dict(lens=lens.long()), "lens"), (dict(table=table[0]), "table"), (dict(cu=cu[:1]), "cu"),
                    (dict(lens=lens.cpu()), "devices"), (dict(q=q[:, :0]), "0 query heads")):
        with pytest.raises(ValueError, match=why):
            attention.chunk_rows(**{**dict(q=q, cache=cache, table=table, lens=lens, cu=cu), **kw})
    with pytest.raises(RuntimeError, match="scale"):
        attention.chunk_rows(q, cache, table, lens, cu, scale=float("nan"))
    assert attention.chunk_rows(q[:0], cache, table, lens, ints([0, 0])).shape == (0, 4, 64)
    assert (attention.chunk_rows(q, cache, table[:0], lens[:0], ints([0])) == 0).all()


def test_serving_run():
    """What a server does with one layer: prompts' chunks (norms of the heads, pages taken, appended, attended), a fork, tokens of
    every sequence with copies of shared pages, a sequence cut, a compaction: against the oracles throughout."""
    from larder_amd import attention, pages as own, trunk
    rng, pick = np.random.default_rng(21), random.Random(21)
    heads, q_heads, width, page, places, count = 2, 6, 64, 32, 8, 60
    cache = attention.KVCache.empty(count, heads, width, page)
    for t in cache:
        t.view(torch.uint8).fill_(0x7f)  # nothing is read that was not written
    refs = torch.zeros(count, dtype=torch.int32, device="cuda")
    table = torch.full((4, places), -1, dtype=torch.int32, device="cuda")
    lens = [0] * 4
    model = ([0] * count, [[-1] * places for _ in range(4)])
    weight = normal(rng, width)
    freq = torch.from_numpy(10000.0 ** (-np.arange(16) / 16)).cuda()

    def step(rows):
        nonlocal model
        for b, r in enumerate(rows):
            lens[b] += r
        cu = cu_of(rows)
        src, dst, lacking = own.take_pages(refs, table, ints(lens), ints(cu), page=page)
        want = pool_ref.take(*model, lens, cu, page)
        model = want[:2]
        assert refs.tolist() == want[0] and table.tolist() == want[1]
        assert src.tolist() == want[2] and dst.tolist() == want[3] and not lacking.any()
        own.copy_pages(cache, src, dst)
        x = normal(rng, cu[-1], q_heads + 2 * heads, width)
        q = trunk.norm_rows(x[:, :q_heads], weight)
        k = trunk.norm_rows(x[:, q_heads:q_heads + heads], weight)
        q, _ = attention.append_rows(cache, q, k, x[:, q_heads + heads:], table, ints(lens), cu=ints(cu), freq=freq)
        got = attention.chunk_rows(q, cache, table, ints(lens), ints(cu))
        check(got, q, cache, np.array(table.tolist()), lens, cu, width ** -0.5, BF16)
        if max(rows) == 1:
            one = attention.attend_rows(q, cache, table, ints(lens), cu=ints(cu))
            check(one, q, cache, np.array(table.tolist()), lens, cu, width ** -0.5, BF16)

    step([40, 0, 65, 3])
    step([20, 33, 30, 64])
    parents = [0, 0, 2, 2, 3, 1]
    new = own.fork_pages(refs, table, ints(parents))
    model = pool_ref.fork(*model, parents)
    assert refs.tolist() == model[0] and new.tolist() == model[1]
    table, lens = new, [lens[p] for p in parents]
    for _ in range(6):
        step([pick.choice([0, 1, 1]) for _ in lens])
    keep = [lens[0], 0, lens[2] - 40, lens[3], 7, lens[5]]
    own.free_pages(refs, table, ints(keep), page=page)
    model = pool_ref.free(*model, keep, page)
    assert refs.tolist() == model[0] and table.tolist() == model[1]
    lens = keep
    step([1, 30, 2, 1, 1, 50])
    src, dst, used = own.compact_pages(refs, table)
    r, t, a, c, u = pool_ref.compact(model[0], [model[1]])
    model = (r, t[0])
    assert refs.tolist() == r and table.tolist() == t[0] and used.tolist() == [u] and src[:len(a)].tolist() == a
    before = attention.read_rows(cache, ints(np.array(src[:len(a)].tolist())[:, None]), ints([page * i for i in range(len(a) + 1)]), page * len(a))
    own.copy_pages(cache, src, dst)
    after = attention.read_rows(cache, dst[:len(c)].view(-1, 1), ints([page * i for i in range(len(c) + 1)]), page * len(c))
    for x, y in zip(before, after):
        assert torch.equal(x.nan_to_num(7.0), y.nan_to_num(7.0))
    assert int(table.max()) < u
    step([5, 1, 1, 40, 1, 1])


def test_trunk_attention_rows_in_chunks():
    """The trunk's call with norms of the heads and chunks over the pages: equal to its parts, a token among them."""
    from larder_amd import attention, trunk
    from test_gpu_attention import affine4
    rng = np.random.default_rng(18)
    hidden, q_heads, heads, width = 512, 4, 1, 128
    qkv, out = affine4(rng, (q_heads + 2 * heads) * width, hidden), affine4(rng, hidden, q_heads * width)
    norms = (normal(rng, width), normal(rng, width), 1e-5)
    freq, _ = attention.rotary_freq(64)
    table = ints([[1, 0, 2]])
    caches = [attention.KVCache.empty(3, heads, width) for _ in range(2)]
    for lens, n, prompt in ((66, 66, "chunk"), (100, 34, "chunk"), (101, 1, None)):
        x, cu = normal(rng, n, hidden), ints([0, n])
        got = trunk.attention_rows(x, qkv, out, caches[0], table, ints([lens]), cu=cu, freq=freq, prompt=prompt, norms=norms)
        q, k, v = trunk.qmv_rows(x, *qkv).view(n, -1, width).split([q_heads, heads, heads], 1)
        q, k = (trunk.norm_rows(y, w, norms[2]) for y, w in zip((q, k), norms))
        q, _ = attention.append_rows(caches[1], q, k, v, table, ints([lens]), cu=cu, freq=freq)
        o = (attention.chunk_rows if prompt else attention.attend_rows)(q, caches[1], table, ints([lens]), cu)
        assert torch.equal(got, trunk.qmv_rows(o.reshape(n, -1), *out))
        check(o, q, caches[1], np.array([[1, 0, 2]]), [lens], [0, n], width ** -0.5, BF16)
    none = trunk.attention_rows(x[:0], qkv, out, caches[0], table, ints([101]), cu=ints([0, 0]), freq=freq, prompt="chunk", norms=norms)
    assert none.shape == (0, hidden)
