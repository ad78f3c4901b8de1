"""GPU parity of the trunk's attention (larder_amd.attention) against the float64 oracle (oracle/attention.py): rotary
positions, appending to the paged 8-bit cache and reading it back, single rows over the cache, whole prompts, and a run of
them together. Caches start poisoned (NaN codes and scales), pages lie in no order.

Tolerances are sums of what the kernels round: half a step of a type (finfo.eps / 2 of the value: bf16 2^-8, fp16 2^-11) each
time a value is rounded to it, and u32 = 2^-24 for float32 arithmetic."""
import numpy as np
import pytest
import torch

from oracle import attention as ref

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def poisoned_memory():
    """What outputs and workspaces are allocated from holds NaN."""
    for n in (1 << 16, 1 << 18, 1 << 22, 1 << 25):
        torch.full((n,), float("nan"), device="cuda")


def host(t):
    return t.detach().double().cpu().numpy()


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def cu_of(lengths):
    return [0] + list(np.cumsum(lengths))


def normal(rng, *shape, dtype=BF16, scale=1.0):
    return torch.from_numpy(rng.standard_normal(shape) * scale).to(dtype).cuda()


def frequencies(pairs):
    return torch.from_numpy(10000.0 ** (-np.arange(pairs) / max(pairs, 1))).cuda()


# ---- rotary positions --------------------------------------------------------------------------------------------

def rope_bound(x, want, freq, gain, dtype):
    """The rounding of the result, and of float32: cos / sin 2 u32 (their argument's rounding and the series'), the gain's
    product, two products and a sum of numbers within |u| + |w|, each u32 of that at most."""
    pair = np.abs(x).max(-1, keepdims=True) * 2 * abs(gain)
    return torch.finfo(dtype).eps / 2 * np.abs(want) + 8 * 2.0 ** -24 * pair + (2.0 ** -25 if dtype == F16 else 0)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("t,heads,width,pairs,interleaved", [
    (1, 32, 128, 64, False), (1, 1, 64, 16, True), (7, 3, 128, 32, False), (3, 5, 256, 32, True), (1500, 4, 64, 32, False),
    (9001, 2, 64, 32, True), (33, 2, 80, 20, False), (33, 2, 90, 9, True), (5, 3, 10, 5, False), (4, 2, 6, 1, True),
    (3, 1, 1024, 512, False), (2, 2, 3, 1, False)])
def test_rope(dtype, t, heads, width, pairs, interleaved):
    from larder_amd import attention
    rng = np.random.default_rng(t + width)
    x = normal(rng, t, heads, width, dtype=dtype)
    pos = torch.from_numpy(rng.integers(-5, 1 << 20, t)).cuda()
    freq = frequencies(pairs)
    gain = 1.0 if t % 2 else 1.25
    got = attention.rope_rows(x, pos, freq, interleaved=interleaved, gain=gain)
    want = ref.rope(host(x), host(pos), host(freq), interleaved, gain)
    assert (np.abs(host(got) - want) <= rope_bound(host(x), want, freq, gain, dtype)).all()
    assert torch.equal(got, attention.rope_rows(x, pos.int(), freq, interleaved=interleaved, gain=gain))
    assert torch.equal(got[..., 2 * pairs:], x[..., 2 * pairs:])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("width,pairs", [(128, 64), (64, 8), (12, 5)])
def test_rope_views_in_place_and_far(interleaved, width, pairs):
    """Views of a wider product and of odd offsets, in place and into a view; a position past 2^53 / 100 turns stays exact."""
    from larder_amd import attention
    rng = np.random.default_rng(4)
    whole = normal(rng, 19, 5, width + 4, dtype=F16)
    x = whole[:, 1:4, 3:3 + width]
    pos = torch.tensor([3 * 10 ** 9] * 19).cuda()
    freq = frequencies(pairs) * 1e-3
    want = attention.rope_rows(x.contiguous(), pos, freq, interleaved=interleaved)
    assert (np.abs(host(want) - ref.rope(host(x), host(pos), host(freq), interleaved)) <=
            rope_bound(host(x), host(want), freq, 1.0, F16) * 1.001).all()
    assert torch.equal(attention.rope_rows(x, pos, freq, interleaved=interleaved), want)
    keep = whole.clone()
    out = torch.full((19, 4, width + 8), 7.0, dtype=F16, device="cuda")
    attention.rope_rows(x, pos, freq, interleaved=interleaved, out=out[:, :3, 8:])
    assert torch.equal(out[:, :3, 8:], want) and (out[:, 3] == 7).all() and (out[:, :, :8] == 7).all()
    assert torch.equal(whole, keep)
    assert attention.rope_rows(x, pos, freq, interleaved=interleaved, out=x) is x
    assert torch.equal(x, want)
    keep[:, 1:4, 3:3 + width] = want
    assert torch.equal(whole, keep)


# ---- the cache ---------------------------------------------------------------------------------------------------

def poisoned(pages, heads, width, page):
    from larder_amd import attention
    c = attention.KVCache.empty(pages, heads, width, page)
    for codes, scales in ((c.k, c.k_scale), (c.v, c.v_scale)):
        codes.view(torch.uint8).fill_(0x7f)
        scales.fill_(float("nan"))
    return c


def cache_host(c):
    return [(a.view(torch.uint8).cpu().numpy().copy(), s.double().cpu().numpy()) for a, s in ((c.k, c.k_scale), (c.v, c.v_scale))]


def page_table(rng, counts, spare=2, width=None):
    n = sum(counts) + spare
    order = rng.permutation(n).astype(np.int32)
    table = np.full((len(counts), width or max(max(counts), 1)), -7, np.int32)
    at = 0
    for b, c in enumerate(counts):
        table[b, :c] = order[at:at + c]
        at += c
    return table, n


def close_codes(got, want, slack):
    """Codes of values that float32 arithmetic moves by at most `slack` (relative to the page's largest): the same value, or
    a neighbour where the exact value lies that close to the middle of the two."""
    a, b = ref.E4M3[got], ref.E4M3[want]
    same = (a == b) | (np.isnan(a) & np.isnan(b))
    step = np.maximum(np.abs(a), np.abs(b)) * 2.0 ** -3 + 2.0 ** -9
    return same.all() or (np.abs(a - b)[~same] <= step[~same] * 1.001).all() and (~same).mean() < slack


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("page,heads,width,pairs,interleaved", [
    (32, 2, 64, 32, False), (64, 4, 128, 64, False), (64, 3, 128, 16, True), (128, 2, 256, 32, False), (128, 1, 256, 128, True),
    (64, 2, 64, 0, False), (32, 1, 256, 128, False)])
def test_append(dtype, page, heads, width, pairs, interleaved):
    """Three calls: ragged prompts (one sequence empty), a second chunk that begins inside pages with larger values, and a token
    each; q, the rotated keys, and every page's codes and scales."""
    from larder_amd import attention
    rng = np.random.default_rng(page + width)
    counts = [[page + 3, 0, 1, 2 * page, page - 1], [5, 2 * page + 1, page, 0, 1], [1, 1, 1, 1, 1]]
    full = np.sum(counts, 0)
    table, n = page_table(rng, [-(-int(x) // page) for x in full])
    cache = poisoned(n, heads, width, page)
    want = cache_host(cache)
    freq = frequencies(pairs) if pairs else None
    lens = np.zeros(5, int)
    for step, new in enumerate(counts):
        lens = lens + new
        cu, t = cu_of(new), sum(new)
        # neighbours in one product, larger values later so that scales grow
        x = normal(rng, t, 3 * heads + 2 * heads, width, dtype=dtype, scale=4.0 ** step)
        q, k, v = x.split([3 * heads, heads, heads], 1)
        got_q, got_k = attention.append_rows(cache, q, k, v, ints(table), ints(lens), cu=ints(cu) if step < 2 else None,
                                             freq=freq, interleaved=interleaved, keys=step != 1)
        pos = np.concatenate([np.arange(m - c, m) for m, c in zip(lens, new)])
        fr = host(freq) if pairs else np.zeros(0)
        for a, b in ((q, got_q), (k, got_k)):
            if b is not None:
                w = ref.rope(host(a), pos, fr, interleaved)
                assert (np.abs(host(b) - w) <= rope_bound(host(a), w, fr, 1.0, dtype)).all()
        assert (got_k is None) == (step == 1)
        ref.append(*want[0], ref.rope(host(k), pos, fr, interleaved), cu, lens, table)
        ref.append(*want[1], host(v), cu, lens, table)
        for (codes, scales), (gc, gs) in zip(want, cache_host(cache)):
            assert np.array_equal(scales, gs, equal_nan=True), step
            # a float32 value off by 8 u32 crosses the middle of two codes (2^-4 of it apart) in about 2^-17 of all cases
            assert close_codes(gc, codes, 1e-4)
            codes[...] = gc  # what later steps restate
        for (codes, scales), tens in zip(want, (cache.k, cache.v)):
            used = np.unique(table[table >= 0])
            rest = np.setdiff1d(np.arange(n), used)
            assert (tens.view(torch.uint8)[torch.from_numpy(rest).cuda()] == 0x7f).all()


@pytest.mark.parametrize("n", [65, 130, 5000])
def test_append_many_sequences(n):
    """More sequences than a wavefront has lanes, and than its square; empty ones among them, one of many rows."""
    from larder_amd import attention
    rng = np.random.default_rng(23)
    rows = [int(x) for x in rng.choice([0, 1, 1, 2], n)]
    rows[n // 2] = 100
    cu = cu_of(rows)
    table, pages = page_table(rng, [-(-x // 32) for x in rows])
    cache = poisoned(pages, 1, 64, 32)
    want = cache_host(cache)
    k, v = (normal(rng, cu[-1], 1, 64) for _ in range(2))
    freq = frequencies(16)
    q, _ = attention.append_rows(cache, k, k, v, ints(table), ints(rows), cu=ints(cu), freq=freq)
    turned = ref.rope(host(k), np.concatenate([np.arange(m) for m in rows]), host(freq))
    assert (np.abs(host(q) - turned) <= rope_bound(host(k), turned, freq, 1.0, BF16)).all()
    ref.append(*want[0], turned, cu, rows, table)
    ref.append(*want[1], host(v), cu, rows, table)
    for (codes, scales), (gc, gs) in zip(want, cache_host(cache)):
        assert np.array_equal(scales, gs, equal_nan=True) and close_codes(gc, codes, 1e-4)
    back, held = attention.read_rows(cache, ints(table), ints(cu), cu[-1], dtype=F32)[0], cache_host(cache)[0]
    want = np.concatenate([ref.read(*held, table[b], rows[b])[0] for b in range(n)])
    assert np.array_equal(host(back), want)


def test_append_token_by_token_and_idempotent():
    """A page filled by single tokens holds what one call writes (values within 2^8 of each other: no code becomes subnormal);
    the same call twice changes nothing."""
    from larder_amd import attention
    rng = np.random.default_rng(8)
    x = torch.from_numpy(rng.uniform(1, 200, (70, 2, 2, 64)) * rng.choice([-1, 1], (70, 2, 2, 64))).to(BF16).cuda()
    k, v = x[:, 0], x[:, 1]
    table = ints([[2, 0]])
    one, grown = poisoned(3, 2, 64, 64), poisoned(3, 2, 64, 64)
    for _ in range(2):
        attention.append_rows(one, None, k, v, table, ints([70]), cu=ints([0, 70]))
        for t in range(70) if _ == 0 else [69]:
            attention.append_rows(grown, None, k[t:t + 1], v[t:t + 1], table, ints([t + 1]))
        for a, b in zip(one, grown):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_append_edges():
    """Values that are not finite, zeros, the smallest scale; pages outside the cache or the table; rows past the last sequence;
    more rows than tokens."""
    from larder_amd import attention
    rng = np.random.default_rng(9)
    k = normal(rng, 12, 1, 64, dtype=F32)
    v = torch.zeros(12, 1, 64, device="cuda")
    k[0, 0, 3], k[0, 0, 4], k[1, 0, 5] = float("nan"), float("inf"), float("-inf")
    v[3, 0, 0], v[3, 0, 1] = 2.0 ** -120, 1e-36
    cache = poisoned(4, 1, 64, 32)
    q, kk = attention.append_rows(cache, k, k, v, ints([[1], [9]]), ints([5, 4]), cu=ints([0, 5, 9]), freq=frequencies(8), keys=True)
    kc, ks = cache_host(cache)[0]
    vc, vs = cache_host(cache)[1]
    want = (np.full((4, 1, 32, 64), 0x7f, np.uint8), np.full((4, 1), np.nan))
    with np.errstate(invalid="ignore"):
        ref.append(*want, ref.rope(host(k), [0, 1, 2, 3, 4] + [0, 1, 2, 3] + [0] * 3, host(frequencies(8))), [0, 5, 9], [5, 4],
                   np.array([[1], [9]]))
    assert np.array_equal(ks, want[1], equal_nan=True) and close_codes(kc, want[0], 1e-3)
    assert np.isnan(ref.E4M3[kc[1, 0, 0]]).sum() >= 2 and (kc[[0, 2, 3]] == 0x7f).all()
    assert vs[1, 0] == 2.0 ** -100 and (vc[1, 0, :5] & 0x7f == 0).all() and np.isnan(vs[[0, 2, 3]]).all()
    assert (q[9:] == 0).all() and (kk[9:] == 0).all() and torch.isfinite(q[5:9]).all()
    # three rows of a sequence of two tokens: the first has no place; a table too short for the rest
    cache = poisoned(4, 1, 64, 32)
    attention.append_rows(cache, None, k[:3], v[:3], ints([[3]]), ints([2]), cu=ints([0, 3]))
    kc = cache_host(cache)[0][0]
    assert close_codes(kc[3, 0, 0], ref.encode_e4m3(host(k[1, 0]) / cache_host(cache)[0][1][3, 0]), 1)
    cache = poisoned(4, 1, 64, 32)
    attention.append_rows(cache, None, k, v, ints([[2]]), ints([38]), cu=ints([0, 12]))
    kc = cache_host(cache)[0][0]
    # the page's held tokens are NaN and stay so, of either sign (their old scale is none)
    assert (kc[2, 0, :26] & 0x7f == 0x7f).all() and not (kc[2, 0, 26:] & 0x7f == 0x7f).all() and (kc[[0, 1, 3]] == 0x7f).all()
    # nothing to do
    q, kk = attention.append_rows(cache, k[:0], k[:0], v[:0], ints([[2]]), ints([38]), cu=ints([0, 0]), freq=frequencies(8))
    assert q.shape == (0, 1, 64) and kk is None


@pytest.mark.parametrize("page,heads,width,rows", [(128, 1, 256, [1500, 3]), (64, 2, 128, [1100, 0, 64]), (32, 1, 64, [8200])])
def test_append_prompts(page, heads, width, rows):
    """Calls of more than 1,024 rows (several rows a rotating workgroup; widest pages: a launch of their own)."""
    from larder_amd import attention
    rng = np.random.default_rng(19)
    cu, t = cu_of(rows), sum(rows)
    table, n = page_table(rng, [-(-x // page) for x in rows])
    cache = poisoned(n, heads, width, page)
    want = cache_host(cache)
    freq = frequencies(width // 4)
    x = normal(rng, t + 1, 4 * heads, width)
    q, k, v = x.split([2 * heads, heads, heads], 1)
    got = attention.append_rows(cache, q, k, v, ints(table), ints(rows), cu=ints(cu), freq=freq, keys=True)
    pos = np.concatenate([np.arange(m) for m in rows] + [[0]])
    for a, b in zip((q, k), got):
        w = ref.rope(host(a), pos, host(freq))
        assert (np.abs(host(b) - w) <= rope_bound(host(a), w, freq, 1.0, BF16))[:t].all() and (b[t:] == 0).all()
    ref.append(*want[0], ref.rope(host(k), pos, host(freq)), cu, rows, table)
    ref.append(*want[1], host(v), cu, rows, table)
    for (codes, scales), (gc, gs) in zip(want, cache_host(cache)):
        assert np.array_equal(scales, gs, equal_nan=True) and close_codes(gc, codes, 1e-4)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("page,heads,width", [(32, 3, 64), (64, 4, 128), (128, 2, 256)])
def test_read(dtype, page, heads, width):
    from larder_amd import attention
    rng = np.random.default_rng(page)
    lens = [3 * page, 0, 1, page + 1, 17]
    table, n = page_table(rng, [-(-x // page) for x in lens])
    cache = random_cache(rng, n, heads, width, page)
    host_cache = cache_host(cache)
    table[3, 1] = n  # a page that is not there
    cu = cu_of(lens)
    k, v = attention.read_rows(cache, ints(table), ints(cu), cu[-1] + 2, dtype=dtype)
    for got, (codes, scales) in zip((k, v), host_cache):
        for b, m in enumerate(lens):
            want, _ = ref.read(codes, scales, table[b], m)
            want = torch.from_numpy(want).to(dtype)
            assert torch.equal(got[cu[b]:cu[b + 1]].cpu(), want)
        assert (got[cu[-1]:] == 0).all()


# ---- single rows over the cache ----------------------------------------------------------------------------------

def random_cache(rng, n, heads, width, page):
    """Every page full of finite codes, scales of several binades."""
    from larder_amd import attention
    c = attention.KVCache.empty(n, heads, width, page)
    for codes, scales in ((c.k, c.k_scale), (c.v, c.v_scale)):
        x = rng.standard_normal((n, heads, page, width)) * 100
        codes.view(torch.uint8).copy_(torch.from_numpy(ref.encode_e4m3(np.clip(x, -448, 448))))
        scales.copy_(torch.from_numpy(np.exp2(rng.integers(-9, -5, (n, heads)))))
    return c


def attention_bound(q, k, scale, out, spread, dtype, weights):
    """The result's rounding; weights rounded to the type `weights` (they stand in the numerator and in the sum it is divided
    by); scores' float32 errors, which change a weight by as much: (width + 8) u32 of sum |q k| scale; exponentials and sums
    2^-19."""
    n, hq, width = q.shape
    g = hq // k.shape[1]
    kk = np.abs(np.where(np.isfinite(k), k, 0)).repeat(g, 1)
    top = np.einsum("ihd,jhd->ihj", np.abs(q), kk).max(-1, initial=0.0)[..., None] * scale
    weight = torch.finfo(weights).eps / 2 + (width + 8) * 2.0 ** -24 * top + 2.0 ** -19
    return torch.finfo(dtype).eps / 2 * np.abs(out) + 2 * weight * spread + (2.0 ** -25 if dtype == F16 else 0) + 1e-30


def check_attend(got, q, cache, table, lens, cu, scale, dtype):
    codes = cache_host(cache)
    qh = host(q)
    for b, n in enumerate(lens):
        x = qh[cu[b]:cu[b + 1]]
        k, there = ref.read(*codes[0], table[b], n)
        v, _ = ref.read(*codes[1], table[b], n)
        want, spread = ref.attend(x, k, v, scale, there)
        have = host(got[cu[b]:cu[b + 1]])
        bound = attention_bound(x, k, scale, want, spread, dtype, F16)
        assert np.array_equal(np.isnan(have), np.isnan(want)), b
        ok = (np.abs(have - want) <= bound) | np.isnan(want)
        assert ok.all(), (b, n, np.abs(have - want)[~ok].max(), bound[~ok].min())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("q_heads,heads,width,page", [(4, 4, 64, 32), (8, 1, 128, 64), (7, 1, 128, 32), (16, 2, 256, 64),
                                                      (40, 2, 64, 128), (3, 3, 256, 128), (12, 4, 128, 128)])
def test_attend(dtype, q_heads, heads, width, page):
    """One row a sequence, lengths of 0, 1, a page's and a tile's ends and odd ones."""
    from larder_amd import attention
    rng = np.random.default_rng(q_heads + width)
    lens = [0, 1, 31, 32, 33, page, page + 1, 3 * page - 1, 500]
    table, n = page_table(rng, [-(-x // page) for x in lens])
    cache = random_cache(rng, n, heads, width, page)
    q = normal(rng, len(lens), q_heads, width, dtype=dtype)
    for longest in (None, 500, 7):
        got = attention.attend_rows(q, cache, ints(table), ints(lens), longest=longest)
        check_attend(got, q, cache, table, lens, list(range(len(lens) + 1)), width ** -0.5, dtype)
        assert torch.equal(got, attention.attend_rows(q, cache, ints(table), ints(lens), longest=longest))
    assert (got[0] == 0).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("q_heads,heads,width,page", [(8, 2, 128, 64), (7, 1, 64, 32), (4, 4, 256, 32), (32, 1, 128, 128)])
def test_attend_draft_rows(dtype, q_heads, heads, width, page):
    """Ragged draft rows (none, one, more than a tile of 16 holds, more than the sequence has tokens), strided, some rows of no
    sequence, launches sized for too few rows and tokens."""
    from larder_amd import attention
    rng = np.random.default_rng(width)
    rows, lens = [5, 0, 1, 19, 4, 3], [300, 64, 97, 40, 2, 0]
    cu = cu_of(rows)
    t = cu[-1] + 2
    table, n = page_table(rng, [-(-x // page) for x in lens])
    cache = random_cache(rng, n, heads, width, page)
    q = normal(rng, t, q_heads + 2, width, dtype=dtype)[:, 1:-1]
    for most, longest in ((19, 300), (1, 1), (None, None), (64, 5000)):
        got = attention.attend_rows(q, cache, ints(table), ints(lens), cu=ints(cu), most_rows=most, longest=longest, scale=0.1)
        check_attend(got, q, cache, table, lens, cu, 0.1, dtype)
        assert (got[cu[-1]:] == 0).all()


@pytest.mark.parametrize("longest", [None, 100])
def test_attend_holes_and_nan(longest):
    """Pages that are not there are not seen; NaN behind the last token or in pages of others is not met, NaN in a seen key or
    value reaches the rows that see it and no other."""
    from larder_amd import attention
    rng = np.random.default_rng(12)
    heads, width, page = 2, 128, 32
    rows, lens = [4, 4, 4, 1], [100, 70, 90, 40]
    cu = cu_of(rows)
    table, n = page_table(rng, [4, 3, 3, 1], width=4)
    table[0, 1], table[0, 2] = -1, 2 ** 31 - 1
    cache = random_cache(rng, n, heads, width, page)
    k, v = cache.k.view(torch.uint8), cache.v.view(torch.uint8)
    for b, m in enumerate(lens):  # behind the last token
        if 0 <= table[b, m // page] < n:
            k[int(table[b, m // page]), :, m % page:] = 0x7f
            v[int(table[b, m // page]), :, m % page:] = 0xff
    v[int(table[1, 2]), 0, 69 - 64, 5] = 0x7f   # the last token of sequence 1: its last row alone
    v[int(table[1, 2]), 1, 68 - 64, 7] = 0xff   # the one before: the last two
    k[int(table[2, 2]), 1, 88 - 64, 9] = 0x7f
    q = normal(rng, cu[-1], 8, width, dtype=F16)
    got = attention.attend_rows(q, cache, ints(table), ints(lens), cu=ints(cu), longest=longest)
    check_attend(got, q, cache, table, lens, cu, width ** -0.5, F16)
    assert torch.isnan(got[7, :4, 5]).all() and not torch.isnan(got[6, :4]).any() and torch.isnan(got[6:8, 4:, 7]).all()
    # a sequence none of whose pages is there
    gone = attention.attend_rows(q, cache, ints(np.full_like(table, n)), ints(lens), cu=ints(cu), longest=longest)
    assert (gone == 0).all()


def test_attend_many_sequences():
    """More sequences than a wavefront has lanes, empty ones and ones longer than their table among them."""
    from larder_amd import attention
    rng = np.random.default_rng(20)
    lens = [int(x) for x in rng.choice([0, 1, 5, 40, 64, 130, 700], 150)]
    lens[7], lens[100] = 2 ** 31 - 1, 900
    rows = [int(x) for x in rng.choice([0, 1, 2], 150)]
    rows[7] = rows[100] = 1
    cu = cu_of(rows)
    table, n = page_table(rng, [min(-(-x // 32), 22) for x in lens], width=22)
    cache = random_cache(rng, n, 1, 64, 32)
    q = normal(rng, cu[-1], 3, 64, dtype=F16)
    got = attention.attend_rows(q, cache, ints(table), ints(lens), cu=ints(cu), longest=704)
    for b in range(150):
        if rows[b]:
            at = slice(cu[b], cu[b + 1])
            check_attend(got[at], q[at], cache, table[b:b + 1], [min(lens[b], 704)], [0, rows[b]], 0.125, F16)
    assert torch.equal(got, attention.attend_rows(q, cache, ints(table), ints(lens), cu=ints(cu), longest=704))


def test_attend_keeps_small_weights():
    """A token that stands out over 8,191 that weigh 2^-20 of it each: together 2^-7, which a float16 weight of 2^-20 would
    lose or move by up to 2^-5 of itself."""
    from larder_amd import attention
    page, n = 64, 128
    cache = attention.KVCache.empty(n, 1, 64, page)
    k, v = torch.zeros(n, 1, page, 64), torch.zeros(n, 1, page, 64)
    k[0, 0, 0, 0], v[..., 1] = 16.0, 1.0
    v[0, 0, 0, 1] = 0.0
    for codes, x in ((cache.k, k), (cache.v, v)):
        codes.view(torch.uint8).copy_(x.to(torch.float8_e4m3fn).view(torch.uint8))
    cache.k_scale.fill_(1.0), cache.v_scale.fill_(1.0)
    q = torch.zeros(1, 1, 64, dtype=F16, device="cuda")
    q[0, 0, 0] = 0.8672  # 20.02 octaves at scale 1
    table, lens = torch.arange(n, dtype=torch.int32, device="cuda")[None], ints([n * page])
    for longest in (None, 128):
        got = attention.attend_rows(q, cache, table, lens, longest=longest, scale=1.0)
        w = (n * page - 1) * np.exp(-16.0 * float(q[0, 0, 0]))
        want = w / (1 + w)
        assert abs(float(got[0, 0, 1]) / want - 1) <= 2.0 ** -11 + 2 * 2.0 ** -11 + 2.0 ** -19, (float(got[0, 0, 1]), want)


def test_offsets_past_32_bits():
    """A cache of more than 2^32 bytes of codes: pages at its end are written, read and attended."""
    from larder_amd import attention
    rng = np.random.default_rng(13)
    page, heads, width = 128, 4, 256
    n = (1 << 32) // (page * heads * width) + 5
    cache = attention.KVCache(*(torch.empty(s, dtype=d, device="cuda") for s, d in
                                (((n, heads, page, width), torch.float8_e4m3fn), ((n, heads), F32)) * 2))
    lens = [200]
    table = np.array([[n - 1, n - 3]], np.int32)
    k, v, q = (normal(rng, 200, h, width, dtype=F16) for h in (heads, heads, 8))
    attention.append_rows(cache, None, k, v, ints(table), ints(lens), cu=ints([0, 200]))
    tail = attention.KVCache(*(t[n - 5:].clone() for t in cache))
    small = table - (n - 5)
    codes = cache_host(tail)
    got = attention.read_rows(cache, ints(table), ints([0, 200]), 200, dtype=F16)
    for x, (c, s), src in zip(got, codes, (k, v)):
        want, _ = ref.read(c, s, small[0], 200)
        assert torch.equal(x.cpu(), torch.from_numpy(want).to(F16))
        assert (np.abs(want - host(src)) <= 2.0 ** -4 * np.abs(host(src)) + 2.0 ** -10 * s[small[0]].max()).all()
    out = attention.attend_rows(q[:1], cache, ints(table), ints(lens))
    check_attend(out, q[:1], tail, small, lens, [0, 1], width ** -0.5, F16)


# ---- whole prompts -----------------------------------------------------------------------------------------------

def check_prompt(got, q, k, v, cu, cu_k, scale, dtype):
    qh, kh, vh = host(q), host(k), host(v)
    for b in range(len(cu) - 1):
        x, y, z = qh[cu[b]:cu[b + 1]], kh[cu_k[b]:cu_k[b + 1]], vh[cu_k[b]:cu_k[b + 1]]
        want, spread = ref.attend(x, y, z, scale)
        have = host(got[cu[b]:cu[b + 1]])
        bound = attention_bound(x, y, scale, want, spread, dtype, dtype)
        assert np.array_equal(np.isnan(have), np.isnan(want)), b
        with np.errstate(invalid="ignore"):
            ok = (np.abs(have - want) <= bound) | np.isnan(want) | (have == want)
        assert ok.all(), (b, np.argwhere(~ok)[:3], np.abs(have - want)[~ok].max(), bound[~ok].min())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("q_heads,heads,width", [(4, 4, 64), (8, 1, 128), (7, 1, 64), (4, 2, 256), (8, 2, 128)])
@pytest.mark.parametrize("lengths", [[1], [129], [64, 1, 0, 63, 65, 128], [300, 31, 0, 0, 200]])
def test_prompt(dtype, q_heads, heads, width, lengths):
    from larder_amd import attention
    rng = np.random.default_rng(sum(lengths) + width)
    cu = cu_of(lengths)
    x = normal(rng, cu[-1] + 1, q_heads + 2 * heads, width, dtype=dtype)  # one row of no sequence
    q, k, v = x.split([q_heads, heads, heads], 1)
    got = attention.prompt_rows(q, k, v, ints(cu))
    check_prompt(got, q, k, v, cu, cu, width ** -0.5, dtype)
    assert (got[cu[-1]:] == 0).all()
    assert torch.equal(got, attention.prompt_rows(q.contiguous(), k.contiguous(), v.contiguous(), ints(cu)))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("width", [64, 128, 256])
def test_prompt_many_sequences(dtype, width):
    """More sequences than a wavefront has lanes, most of them a row or none."""
    from larder_amd import attention
    rng = np.random.default_rng(22)
    lengths = [int(x) for x in rng.choice([0, 0, 1, 2, 9], 300)]
    lengths[17], lengths[299] = 140, 0
    cu = cu_of(lengths)
    q, k, v = normal(rng, cu[-1] + 1, 2, width, dtype=dtype), *(normal(rng, cu[-1] + 1, 1, width, dtype=dtype) for _ in range(2))
    got = attention.prompt_rows(q, k, v, ints(cu))
    check_prompt(got, q, k, v, cu, cu, width ** -0.5, dtype)
    assert (got[cu[-1]:] == 0).all()


@pytest.mark.parametrize("lengths", [[128] * 70, [127, 129] * 33, [1] * 64 + [300, 256, 384]])
def test_prompt_many_full_tiles(lengths):
    """More sequences than a wavefront has lanes, whose rows fill their tiles or just do not: every tile is worked once."""
    from larder_amd import attention
    rng = np.random.default_rng(len(lengths))
    cu = cu_of(lengths)
    q, k, v = normal(rng, cu[-1], 2, 64, dtype=F16), *(normal(rng, cu[-1], 1, 64, dtype=F16) for _ in range(2))
    check_prompt(attention.prompt_rows(q, k, v, ints(cu)), q, k, v, cu, cu, 64 ** -0.5, F16)


@pytest.mark.parametrize("width", [64, 128, 256])
def test_prompt_rows_far_apart(width):
    """Query rows whose strides pass 2^31 bytes together, and a page-long gap between keys."""
    from larder_amd import attention
    rng = np.random.default_rng(width + 1)
    wide = torch.zeros(40, 2 ** 24 + 8, dtype=F16, device="cuda")
    q = wide[:, :2 * width].view(40, 2, width)
    q.copy_(normal(rng, 40, 2, width, dtype=F16))
    k, v = (normal(rng, 40, 40, width, dtype=F16)[:, 7:8] for _ in range(2))
    got = attention.prompt_rows(q, k, v, ints([0, 40]))
    assert torch.equal(got, attention.prompt_rows(q.contiguous(), k.contiguous(), v.contiguous(), ints([0, 40])))
    check_prompt(got, q, k, v, [0, 40], [0, 40], width ** -0.5, F16)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("width", [64, 128, 256])
def test_prompt_over_more_and_fewer_keys(dtype, width):
    """Chunks over a history, and sequences with fewer keys than rows, whose first rows see none."""
    from larder_amd import attention
    rng = np.random.default_rng(width)
    rows, keys = [100, 7, 150, 40, 3], [391, 7, 20, 0, 1000]
    cu, cu_k = cu_of(rows), cu_of(keys)
    q, k, v = normal(rng, cu[-1], 6, width, dtype=dtype), *(normal(rng, cu_k[-1], 3, width, dtype=dtype) for _ in range(2))
    got = attention.prompt_rows(q, k, v, ints(cu), cu_k=ints(cu_k), scale=0.2)
    check_prompt(got, q, k, v, cu, cu_k, 0.2, dtype)
    assert (got[cu[2]:cu[2] + 130] == 0).all() and (got[cu[3]:cu[4]] == 0).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("width", [64, 128, 256])
@pytest.mark.parametrize("rows,keys", [([100], [3000]), ([130, 1, 200], [1300, 2200, 200]), ([5, 5], [0, 0])])
def test_prompt_keys_in_chunks(dtype, width, rows, keys):
    """Few rows over many keys: the keys go to several workgroups; no keys at all."""
    from larder_amd import _lib, attention
    rng = np.random.default_rng(sum(keys) + width)
    cu, cu_k = cu_of(rows), cu_of(keys)
    q, k, v = normal(rng, cu[-1] + 2, 4, width, dtype=dtype), *(normal(rng, cu_k[-1], 2, width, dtype=dtype) for _ in range(2))
    split = _lib.lib().lmoe_prompt_attend_workspace_bytes(q.shape[0], k.shape[0], 4, 2, width, len(rows))
    assert (split > 0) == (sum(keys) > 0)
    got = attention.prompt_rows(q, k, v, ints(cu), cu_k=ints(cu_k))
    check_prompt(got, q, k, v, cu, cu_k, width ** -0.5, dtype)
    assert (got[cu[-1]:] == 0).all() and torch.equal(got, attention.prompt_rows(q, k, v, ints(cu), cu_k=ints(cu_k)))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("width", [64, 128, 256])
def test_prompt_values_not_finite(dtype, width):
    """NaN and infinities in values and keys reach the rows that see them, and no row before or other sequence."""
    from larder_amd import attention
    rng = np.random.default_rng(14)
    lengths = [150, 70, 40]
    cu = cu_of(lengths)
    q, k, v = (normal(rng, cu[-1], h, width, dtype=dtype) for h in (2, 1, 1))
    clean = attention.prompt_rows(q, k, v, ints(cu))
    v[100, 0, 3], v[140, 0, 4], v[149, 0, 5] = float("nan"), float("inf"), float("-inf")
    v[150, 0, 6] = float("inf")
    k[219, 0, 0] = float("nan")
    got = attention.prompt_rows(q, k, v, ints(cu))
    assert torch.equal(got[:100], clean[:100]) and torch.isnan(got[100:150, :, 3]).all()
    assert (got[140:150, :, 4] == float("inf")).all() and (got[149, :, 5] == float("-inf")).all()
    assert torch.isfinite(got[100:140, :, 4:]).all() and torch.isfinite(got[:149, :, 5]).all()
    assert (got[150:219, :, 6] == float("inf")).all() and torch.isnan(got[219]).all()
    assert torch.equal(got[220:], clean[220:])
    check_prompt(got[:100], q[:100], k[:100], v[:100], [0, 100], [0, 100], width ** -0.5, dtype)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("width,rows,keys", [(64, 130, 130), (128, 40, 2100), (256, 70, 70)])
def test_prompt_scores_of_minus_infinity(dtype, width, rows, keys):
    """Keys whose scores are -inf weigh nothing, in whole tiles and chunks and among others; a row with only such is zero."""
    from larder_amd import attention
    rng = np.random.default_rng(16)
    q, k, v = (normal(rng, n, 1, width, dtype=dtype) for n in (rows, keys, keys))
    q[:, 0, 0] = q[:, 0, 0].abs() + 1
    k[:keys - rows + 20, 0, 0] = float("-inf")
    k[keys - 10, 0, 0] = float("-inf")
    got = attention.prompt_rows(q, k, v, ints([0, rows]), cu_k=ints([0, keys]))
    assert (got[:20] == 0).all() and (got[20:] != 0).any(-1).all()
    check_prompt(got, q, k, v, [0, rows], [0, keys], width ** -0.5, dtype)


def test_attend_scores_of_minus_infinity():
    """A query that scores -inf against every token (or all but those of one page) among others that do not."""
    from larder_amd import attention
    rng = np.random.default_rng(17)
    cache = random_cache(rng, 30, 1, 64, 64)
    codes = cache.k.view(torch.uint8)
    codes[:, :, :, 0] = 0x38   # 1.0
    codes[29, :, :, 0] = 0xb8  # -1.0: +inf against the second query, which is NaN
    table, lens = np.arange(30, dtype=np.int32)[None].repeat(3, 0), np.array([29 * 64, 30 * 64, 29 * 64 - 5], np.int32)
    q = normal(rng, 3, 2, 64, dtype=F16)
    q[:2, 0, 0] = float("-inf")
    for longest in (None, 1):
        got = attention.attend_rows(q, cache, ints(table), ints(lens), longest=longest)
        assert (got[0, 0] == 0).all() and torch.isnan(got[1, 0]).all() and torch.isfinite(got[2]).all()
        check_attend(got[2:], q[2:], cache, table[2:], lens[2:], [0, 1], 64 ** -0.5, F16)
        check_attend(got[:1, 1:], q[:1, 1:], cache, table, lens[:1], [0, 1], 64 ** -0.5, F16)


def test_large_scores():
    """Scores in the thousands, one key far above the rest, and equal scores: no overflow, the weights of a softmax."""
    from larder_amd import attention
    rng = np.random.default_rng(15)
    q, k, v = (normal(rng, 200, h, 128, dtype=BF16, scale=s) for h, s in ((4, 30), (2, 30), (2, 1)))
    got = attention.prompt_rows(q, k, v, ints([0, 200]))
    assert torch.isfinite(got).all()
    same = attention.prompt_rows(q * 0, k, v, ints([0, 200]))
    want = torch.cumsum(v.double(), 0) / torch.arange(1, 201, device="cuda")[:, None, None]
    want = want.repeat_interleave(2, 1)
    # equal weights are exact: the float32 sums' and the result's rounding are left
    assert ((same.double() - want).abs() <= want.abs() * 2.0 ** -8 + 2.0 ** -15).all()


# ---- together ----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,q_heads,heads,width,page", [(BF16, 8, 2, 128, 64), (F16, 4, 1, 256, 32)])
def test_chunked_prompt_then_tokens(dtype, q_heads, heads, width, page):
    """Two prompts in two chunks each, then tokens one by one: every output against float64 attention over what the cache
    holds (its own values for the first chunk, whose attention reads the rows themselves)."""
    from larder_amd import attention
    rng = np.random.default_rng(16)
    freq, gain = attention.rotary_freq(width // 2, 1e6, "yarn", 4.0, 4096)
    chunks, steps = [[70, 33], [50, 100]], 3
    total = [sum(c) + steps for c in zip(*chunks)]
    table, n = page_table(rng, [-(-x // page) for x in total])
    cache, dev_table = poisoned(n, heads, width, page), ints(table)
    lens = np.zeros(2, int)
    for step, new in enumerate(chunks + [[1, 1]] * steps):
        lens, cu = lens + new, cu_of(new)
        x = normal(rng, cu[-1], q_heads + 2 * heads, width, dtype=dtype)
        q, k, v = x.split([q_heads, heads, heads], 1)
        q, k = attention.append_rows(cache, q, k, v, dev_table, ints(lens), cu=ints(cu), freq=freq, gain=gain, keys=step == 0)
        if step == 0:
            out = attention.prompt_rows(q, k, v, ints(cu))
            check_prompt(out, q, k, v, cu, cu, width ** -0.5, dtype)
        elif step == 1:
            cu_k = cu_of(lens)
            hk, hv = attention.read_rows(cache, dev_table, ints(cu_k), cu_k[-1], dtype=dtype)
            out = attention.prompt_rows(q, hk, hv, ints(cu), cu_k=ints(cu_k))
            check_prompt(out, q, hk, hv, cu, cu_k, width ** -0.5, dtype)
        else:
            out = attention.attend_rows(q, cache, dev_table, ints(lens), cu=ints(cu))
            check_attend(out, q, cache, table, lens, cu, width ** -0.5, dtype)


def test_decode_step_in_a_graph():
    """append and attend captured once and replayed while lens, the rows and the cache move on: each replay equals the eager
    calls on a second cache."""
    from larder_amd import attention
    rng = np.random.default_rng(17)
    heads, width, page, batch = 2, 128, 64, 3
    table = ints(rng.permutation(12).reshape(3, 4))
    lens = ints([60, 1, 130])
    eager, caught = (attention.KVCache.empty(12, heads, width, page) for _ in range(2))
    past = [normal(rng, 191, heads, width) for _ in range(2)]
    for c in (eager, caught):
        attention.append_rows(c, None, *past, table, lens, cu=ints([0, 60, 61, 191]))
    freq, _ = attention.rotary_freq(width)
    x = normal(rng, batch, 8 + 2 * heads, width)

    def step(c):
        q, k, v = x.split([8, heads, heads], 1)
        q, _ = attention.append_rows(c, q, k, v, table, lens, freq=freq)
        return attention.attend_rows(q, c, table, lens, longest=256)
    lens += 1
    want = step(eager)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(step(caught), want)  # a warm-up, on another stream than the default
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(caught)
    for i in range(6):
        lens += 1
        x.copy_(normal(rng, batch, 8 + 2 * heads, width, scale=1.0 + i))
        want = step(eager)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
        for a, b in zip(eager, caught):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("width", [128, 256])
def test_prompt_in_a_graph_and_on_streams(width):
    """A prompt chunk (keys in chunks, their workspace in the graph's memory) replayed between eager calls, and two calls on two
    streams at once."""
    from larder_amd import attention
    rng = np.random.default_rng(21)
    q, k, v = normal(rng, 70, 4, width), normal(rng, 2000, 2, width), normal(rng, 2000, 2, width)
    cu, cu_k = ints([0, 70]), ints([0, 2000])
    cache = attention.KVCache.empty(40, 2, width)
    table, lens = torch.arange(40, dtype=torch.int32, device="cuda")[None], ints([2000])
    attention.append_rows(cache, None, k, v, table, lens, cu=cu_k)

    def both():
        return attention.prompt_rows(q, k, v, cu, cu_k=cu_k), attention.attend_rows(q[:3], cache, table, lens, cu=ints3)
    ints3 = ints([0, 3])
    both()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        caught = both()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for i in range(4):
        q.copy_(normal(rng, 70, 4, width))
        want = both()
        g.replay()
        torch.cuda.synchronize()
        outs = []
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(both())
        torch.cuda.synchronize()
        for got in [caught] + outs:
            assert all(torch.equal(a, b) for a, b in zip(got, want)), i


def test_trunk_attention_rows():
    """The trunk's call on 4-bit projections: a prompt, a second chunk over the cache, a token; equal to its parts."""
    from larder_amd import attention, trunk
    from oracle import qmv
    rng = np.random.default_rng(18)
    H, q_heads, heads, width, G = 512, 4, 1, 128, 64

    def weight(n, k):
        wq, s, b = qmv.quantize_affine4((rng.standard_normal((n, k)) * 0.05).astype(np.float32), G)
        return torch.from_numpy(wq.view(np.int32)).cuda(), *(torch.from_numpy(np.ascontiguousarray(a)).cuda().bfloat16() for a in (s, b)), G
    qkv, out = weight((q_heads + 2 * heads) * width, H), weight(H, q_heads * width)
    freq, gain = attention.rotary_freq(64)
    table = ints([[1, 0, 2]])
    caches = [attention.KVCache.empty(3, heads, width) for _ in range(2)]
    for lens, n, prompt in ((66, 66, True), (100, 34, "history"), (101, 1, None)):
        x, cu = normal(rng, n, H), ints([0, n])
        kind = (ints([0, lens]), lens) if prompt == "history" else prompt
        got = trunk.attention_rows(x, qkv, out, caches[0], table, ints([lens]), cu=cu, freq=freq, gain=gain, prompt=kind)
        q, k, v = trunk.qmv_rows(x, *qkv).view(n, -1, width).split([q_heads, heads, heads], 1)
        q, k = attention.append_rows(caches[1], q, k, v, table, ints([lens]), cu=cu, freq=freq, gain=gain, keys=True)
        if prompt is True:
            o = attention.prompt_rows(q, k, v, cu)
        elif prompt:
            o = attention.prompt_rows(q, *attention.read_rows(caches[1], table, kind[0], lens), cu, cu_k=kind[0])
        else:
            o = attention.attend_rows(q, caches[1], table, ints([lens]))
        assert torch.equal(got, trunk.qmv_rows(o.reshape(n, -1), *out))
        assert torch.isfinite(got).all() and float(got.float().std()) > 0
    with pytest.raises(ValueError, match="offsets"):
        trunk.attention_rows(x, qkv, out, caches[0], table, ints([101]), prompt=True)
    with pytest.raises(ValueError, match="heads"):
        trunk.attention_rows(x, weight(2 * width, H), out, caches[0], table, ints([101]))


def test_refusals():
    from larder_amd import attention
    q = torch.zeros(2, 4, 128, dtype=F16, device="cuda")
    k = torch.zeros(2, 2, 128, dtype=F16, device="cuda")
    cache, table, lens, cu = attention.KVCache.empty(2, 2, 128), ints([[0], [1]]), ints([1, 1]), ints([0, 1, 2])
    freq = frequencies(64)
    for bad in (lambda: attention.attend_rows(q.float(), cache, table, lens),
                lambda: attention.attend_rows(q[:, :3], cache, table, lens),
                lambda: attention.attend_rows(q[:1], cache, table, lens),
                lambda: attention.attend_rows(q, cache, table.long(), lens),
                lambda: attention.attend_rows(q, cache, table, lens.cpu()),
                lambda: attention.attend_rows(q, cache, table, lens[:1]),
                lambda: attention.attend_rows(q, cache._replace(k_scale=cache.k_scale.half()), table, lens),
                lambda: attention.attend_rows(q, cache._replace(k=cache.k.transpose(0, 1), v=cache.v.transpose(0, 1)), table, lens),
                lambda: attention.attend_rows(q[..., :64], cache, table, lens),
                lambda: attention.append_rows(cache, q, k, k.bfloat16(), table, lens),
                lambda: attention.append_rows(cache, q, k, k[:1], table, lens),
                lambda: attention.append_rows(cache, q, k[:, :1], k, table, lens),
                lambda: attention.append_rows(cache, q, k, k, table, lens, freq=freq.float()),
                lambda: attention.append_rows(cache, q, k, k, table, lens, cu=cu[:2]),
                lambda: attention.read_rows(cache, table, None, 2),
                lambda: attention.read_rows(cache, table, cu, 2, dtype=torch.int32),
                lambda: attention.prompt_rows(q, k, k, cu.long()),
                lambda: attention.prompt_rows(q, k[:1], k[:1], cu),
                lambda: attention.prompt_rows(q, k, k.bfloat16(), cu),
                lambda: attention.prompt_rows(q.float(), k.float(), k.float(), cu),
                lambda: attention.prompt_rows(q[..., :32], k[..., :32], k[..., :32], cu),
                lambda: attention.rope_rows(q, lens.float(), freq),
                lambda: attention.rope_rows(q, lens[:1], freq),
                lambda: attention.rope_rows(q, lens, frequencies(65)),
                lambda: attention.rope_rows(q.double(), lens, freq),
                lambda: attention.rope_rows(q, lens, freq, out=q.bfloat16()),
                lambda: attention.KVCache.empty(2, 2, 96), lambda: attention.KVCache.empty(2, 2, 64, page=16)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="pairs"):
        attention.append_rows(cache, q, k, k, table, lens, freq=frequencies(10))
    odd = torch.zeros(2 * 512 + 1, dtype=F16, device="cuda")[1:].view(2, 4, 128)  # rows at odd addresses are copied, not refused
    assert torch.equal(attention.attend_rows(odd, cache, table, lens), attention.attend_rows(q, cache, table, lens))


@pytest.mark.parametrize("width,page", [(64, 32), (128, 64), (256, 64)])
def test_one_row_or_head_with_a_stride_of_its_own(width, page):
    """A single row out of a padded product, and a single head with an odd head stride: appended, attended and run as a prompt as
    their dense copies are."""
    from larder_amd import attention
    rng = np.random.default_rng(width)
    padded = normal(rng, 9, 4 * width + 3)
    row = padded[:, :4 * width].view(9, 4, width)[3:4]                 # row stride 4 width + 3
    head = normal(rng, 5, 3, width + 1)[2:3, 1:2, 1:]                  # head stride width + 1, an odd address
    q, k, v = row[:, :2], row[:, 2:3], head
    assert q.stride(0) % 8 and k.stride(0) % 8 and v.stride(1) % 8
    table, lens, freq = ints([[1]]), ints([1]), frequencies(16)
    outs = []
    for a, b, c in ((q, k, v), (q.clone(memory_format=torch.contiguous_format).reshape(-1).view(1, 2, width),
                                k.reshape(-1).view(1, 1, width).clone(), v.reshape(-1).view(1, 1, width).clone())):
        cache = poisoned(2, 1, width, page)
        turned, keys = attention.append_rows(cache, a, b, c, table, lens, freq=freq, keys=True)
        outs.append([turned, keys, *(t.view(torch.uint8) for t in cache), attention.attend_rows(a, cache, table, lens),
                     attention.prompt_rows(a, b, c, ints([0, 1]))])
    for x, y in zip(*outs):
        assert torch.equal(x, y)
    check_prompt(outs[0][-1], q, k, v, [0, 1], [0, 1], width ** -0.5, BF16)


def test_prompt_keys_far_apart():
    """Keys and values of rows 2^23 elements and more apart, and one key of such rows."""
    from larder_amd import attention
    rng = np.random.default_rng(31)
    wide = torch.zeros(5, (1 << 23) + 8, dtype=F16, device="cuda")
    wide[:, :512] = normal(rng, 5, 512, dtype=F16)
    q, k, v = normal(rng, 5, 4, 128, dtype=F16), wide[:, :256].view(5, 2, 128), wide[:, 256:512].view(5, 2, 128)
    for n in (5, 1):
        got = attention.prompt_rows(q[:n], k[:n], v[:n], ints([0, n]))
        check_prompt(got, q[:n], k[:n], v[:n], [0, n], [0, n], 128 ** -0.5, F16)


def affine4(rng, n, k, group=64):
    """A 4-bit affine weight [n, k] for trunk.qmv_rows."""
    from oracle import qmv
    wq, s, b = qmv.quantize_affine4((rng.standard_normal((n, k)) * 0.05).astype(np.float32), group)
    return torch.from_numpy(wq.view(np.int32)).cuda(), *(torch.from_numpy(np.ascontiguousarray(a)).cuda().bfloat16() for a in (s, b)), group


def test_trunk_attention_refuses_before_it_writes():
    """Refused calls of attention_rows leave the cache as it was."""
    from larder_amd import trunk
    rng = np.random.default_rng(32)
    cache = random_cache(rng, 2, 2, 64, 32)
    before = [t.clone() for t in cache]
    x, qkv, out = normal(rng, 1, 128), affine4(rng, 8 * 64, 128), affine4(rng, 128, 4 * 64)
    table, lens, cu = ints([[0]]), ints([1]), ints([0, 1])
    for kw, why in ((dict(prompt=(cu, 1)), "offsets"), (dict(prompt=(cu.cpu(), 1), cu=cu), "lives"),
                    (dict(qkv=affine4(rng, 7 * 64, 128)), "heads"), (dict(out=affine4(rng, 128, 3 * 64)), "out")):
        with pytest.raises(ValueError, match=why):
            trunk.attention_rows(x, **{**dict(qkv=qkv, out=out, cache=cache, table=table, lens=lens), **kw})
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(cache, before))


def test_trunk_attention_of_no_rows():
    """A call without rows gives none back, and changes no page."""
    from larder_amd import trunk
    rng = np.random.default_rng(33)
    cache = random_cache(rng, 2, 2, 64, 32)
    before = [t.clone() for t in cache]
    qkv, out, cu = affine4(rng, 8 * 64, 128), affine4(rng, 128, 4 * 64), ints([0, 0])
    for prompt in (None, True, (ints([0, 5]), 5)):
        got = trunk.attention_rows(normal(rng, 0, 128), qkv, out, cache, ints([[1]]), ints([5]), cu=cu, prompt=prompt)
        assert got.shape == (0, 128) and got.dtype == BF16
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(cache, before))


@pytest.mark.parametrize("rotated", [False, True])
@pytest.mark.parametrize("rows", [[3, 0, 2], [1200, 40, 1], [0, 0, 0]])
def test_append_rows_of_no_sequence_come_back_zero(rows, rotated):
    """Rows before the first sequence and behind the last one, with a rotation and without, and a call of no sequences."""
    from larder_amd import attention
    rng = np.random.default_rng(34)
    cu = [2 + int(x) for x in cu_of(rows)]
    t = cu[-1] + 3
    x = normal(rng, t, 4, 64)
    q, k, v = x.split([2, 1, 1], 1)
    table, n = page_table(rng, [-(-m // 32) for m in rows])
    freq = frequencies(16) if rotated else None
    got = attention.append_rows(poisoned(n, 1, 64, 32), q, k, v, ints(table), ints(rows), cu=ints(cu), freq=freq, keys=True)
    pos = np.concatenate([np.zeros(2, int)] + [np.arange(m) for m in rows] + [np.zeros(3, int)])
    for a, b in zip((q, k), got):
        assert (b[:2] == 0).all() and (b[cu[-1]:] == 0).all()
        w = ref.rope(host(a), pos, host(freq) if rotated else [])
        assert (np.abs(host(b) - w) <= rope_bound(host(a), w, freq, 1.0, BF16))[2:cu[-1]].all()
        assert rotated or torch.equal(b[2:cu[-1]], a[2:cu[-1]])
    none = attention.append_rows(poisoned(n, 1, 64, 32), q, k, v, ints(table)[:0], ints(rows)[:0], cu=ints([2]), freq=freq, keys=True)
    assert all((a == 0).all() for a in none) and (x != 0).any()


def test_append_gives_tensors_of_its_own():
    """Writing to what append_rows returned does not reach the caller's q and k, with a rotation or without."""
    from larder_amd import attention
    x = torch.ones(1, 4, 64, dtype=F16, device="cuda")
    for freq in (None, frequencies(0), frequencies(8)):
        cache = attention.KVCache.empty(1, 1, 64)
        q, k = attention.append_rows(cache, x[:, :2], x[:, 2:3], x[:, 3:], ints([[0]]), ints([1]), freq=freq, keys=True)
        q.zero_(), k.zero_()
        assert (x == 1).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_history_with_holes_read_without_them(dtype):
    """A prompt chunk over a history some of whose pages are gone: attend_rows through the table with the holes, and prompt_rows
    over what a table without them reads, are the same attention."""
    from larder_amd import attention
    rng = np.random.default_rng(35)
    heads, width, page = 2, 128, 32
    rows, lens = [9, 20], [150, 70]
    cu = cu_of(rows)
    table, n = page_table(rng, [5, 3])
    cache = random_cache(rng, n, heads, width, page)
    held = [table[0][[0, 3, 4]], table[1][[1, 2]]]
    gaps = table.copy()
    gaps[0, 1], gaps[0, 2], gaps[1, 0] = -1, n, -5
    compact = np.full((2, 3), -1, np.int32)
    compact[0], compact[1, :2] = held
    cu_k = cu_of([150 - 64, 70 - 32])
    q = normal(rng, cu[-1], 4, width, dtype=dtype)
    over_cache = attention.attend_rows(q, cache, ints(gaps), ints(lens), cu=ints(cu))
    check_attend(over_cache, q, cache, gaps, lens, cu, width ** -0.5, dtype)
    k, v = attention.read_rows(cache, ints(compact), ints(cu_k), cu_k[-1], dtype=dtype)
    over_rows = attention.prompt_rows(q, k, v, ints(cu), cu_k=ints(cu_k))
    for b in range(2):
        codes = cache_host(cache)
        (hk, there), (hv, _) = (ref.read(*c, gaps[b], lens[b]) for c in codes)
        x, have = host(q[cu[b]:cu[b + 1]]), host(over_rows[cu[b]:cu[b + 1]])
        want, spread = ref.attend(x, hk, hv, width ** -0.5, there)
        assert (np.abs(have - want) <= attention_bound(x, hk, width ** -0.5, want, spread, dtype, dtype)).all()


# ---- larger sizes, and a page's codes whatever begins it ---------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("q_heads,heads,width,rows,keys", [
    (2, 1, 64, [1500], [1500]), (2, 1, 128, [1031, 640], [1031, 640]), (2, 2, 256, [900], [900]), (2, 1, 128, [700], [2900]),
    (1, 1, 64, [513] * 2 + [1] * 70, [513] * 2 + [1] * 70)])
def test_prompt_long(dtype, q_heads, heads, width, rows, keys):
    """Prompts of many tiles, alone, beside others and over a history: the loop's full tiles, between its first and last."""
    from larder_amd import attention
    rng = np.random.default_rng(sum(rows) + width)
    cu, cu_k = cu_of(rows), cu_of(keys)
    q, k, v = normal(rng, cu[-1], q_heads, width, dtype=dtype), *(normal(rng, cu_k[-1], heads, width, dtype=dtype) for _ in range(2))
    got = attention.prompt_rows(q, k, v, ints(cu), cu_k=ints(cu_k))
    check_prompt(got, q, k, v, cu, cu_k, width ** -0.5, dtype)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("q_heads,heads,width,page,rows,lens", [
    (7, 1, 128, 64, [1], [9001]), (4, 2, 64, 128, [1, 1, 1], [5000, 12, 7777]), (4, 1, 256, 32, [1, 3], [4100, 2500]),
    (8, 1, 128, 64, [16], [6000]), (8, 2, 64, 32, [16, 5], [3500, 2101])])
def test_attend_long(dtype, q_heads, heads, width, page, rows, lens):
    """Long caches of varied values: many units an item, joined from several workgroups; single and draft rows."""
    from larder_amd import attention
    rng = np.random.default_rng(sum(lens))
    cu = cu_of(rows)
    table, n = page_table(rng, [-(-x // page) for x in lens])
    cache = random_cache(rng, n, heads, width, page)
    q = normal(rng, cu[-1], q_heads, width, dtype=dtype)
    for longest in (None, max(lens), 600):
        got = attention.attend_rows(q, cache, ints(table), ints(lens), cu=ints(cu), most_rows=max(rows), longest=longest)
        check_attend(got, q, cache, table, lens, cu, width ** -0.5, dtype)


@pytest.mark.parametrize("rows,tokens", [(3, 2), (40, 33), (5, 1), (4, 0)])
def test_append_more_rows_than_tokens(rows, tokens):
    """Rows that stand before a sequence's first place are not written; the page's whole codes and its scale are those of the
    tokens that have a place."""
    from larder_amd import attention
    rng = np.random.default_rng(rows)
    k, v = (normal(rng, rows, 2, 64, dtype=F32, scale=s) for s in (1, 9))
    k[0], v[0] = 1e6, 1e6  # before the first place: not in the scale
    cache, table = poisoned(4, 2, 64, 32), np.array([[3, 1]])
    want = cache_host(cache)
    attention.append_rows(cache, None, k, v, ints(table), ints([tokens]), cu=ints([0, rows]))
    for (codes, scales), x in zip(want, (k, v)):
        ref.append(codes, scales, host(x)[rows - tokens:], [0, tokens], [tokens], table)
    for (codes, scales), (gc, gs) in zip(want, cache_host(cache)):
        assert np.array_equal(scales, gs, equal_nan=True)
        assert np.array_equal(codes & 0x7f == 0x7f, gc & 0x7f == 0x7f) and np.array_equal(
            np.nan_to_num(ref.E4M3[codes]), np.nan_to_num(ref.E4M3[gc]))  # no rotation: powers of two, one rounding, exactly


def test_trunk_attention_against_float64():
    """attention_rows against float64 from its 4-bit products on: a prompt, a later chunk, draft rows, a token, with a rotation of
    half a head. The output weight is the identity (values 0 and 1, scale 1, no bias), which qmv gives back exactly, and the
    products before it are the oracle's bits. q, and in the first chunk k, are rounded to bfloat16 once more than the oracle's:
    each moves a score by 2^-8 of sum |q k| scale at most, and a weight by as much of itself, in a row's sums twice."""
    from larder_amd import attention, trunk
    from oracle import qmv
    rng = np.random.default_rng(36)
    H, q_heads, heads, width, G = 256, 4, 2, 64, 64
    rows = (q_heads + 2 * heads) * width
    wq, sc, bi = qmv.quantize_affine4((rng.standard_normal((rows, H)) * 0.05).astype(np.float32), G)
    one = np.zeros((q_heads * width, q_heads * width // 8), np.uint32)
    for i in range(q_heads * width):
        one[i, i // 8] = 1 << 4 * (i % 8)
    ones = np.ones((q_heads * width, q_heads * width // G), np.float32)
    x0 = qmv.bf16(rng.standard_normal((2, q_heads * width)))
    assert np.array_equal(qmv.qmv_rows(x0, one, ones, 0 * ones, G), x0)

    def dev(w, s, b):
        return torch.from_numpy(w.view(np.int32)).cuda(), *(torch.from_numpy(np.ascontiguousarray(a, np.float32)).cuda().bfloat16()
                                                           for a in (s, b)), G
    qkv, out = dev(wq, sc, bi), dev(one, ones, 0 * ones)
    freq, gain = attention.rotary_freq(32, 1e4, "linear", 2.0)
    table, n = page_table(rng, [5, 4])
    cache, lens = poisoned(n, heads, width, 32), np.zeros(2, int)
    for new, kind in (([70, 41], "first"), ([30, 50], "later"), ([3, 1], "drafts"), ([1, 1], "token")):
        lens, cu = lens + new, cu_of(new)
        x = normal(rng, cu[-1], H)
        cu_k = cu_of(lens)
        got = trunk.attention_rows(x, qkv, out, cache, ints(table), ints(lens), cu=None if kind == "token" else ints(cu), freq=freq,
                                   gain=gain, prompt={"first": True, "later": (ints(cu_k), cu_k[-1])}.get(kind),
                                   most_rows=3 if kind == "drafts" else None)
        y = qmv.qmv_rows(host(x).astype(np.float32), wq, sc, bi, G).astype(np.float64).reshape(cu[-1], -1, width)
        codes = cache_host(cache)
        for b in range(2):
            at, pos = slice(cu[b], cu[b + 1]), np.arange(lens[b] - new[b], lens[b])
            q, k = (ref.rope(y[at, h], pos, host(freq), False, gain) for h in (slice(q_heads), slice(q_heads, q_heads + heads)))
            v = y[at, q_heads + heads:]
            if kind != "first":
                k, v = (ref.read(*c, table[b], lens[b])[0] for c in codes)
            want, spread = ref.attend(q, k, v, width ** -0.5)
            top = np.einsum("ihd,jhd->ihj", np.abs(q), np.abs(k).repeat(2, 1)).max(-1)[..., None] * width ** -0.5
            moved = 2 * (2 if kind == "first" else 1) * 2.0 ** -8 * top * 1.01
            bound = attention_bound(q, k, width ** -0.5, want, spread, BF16, BF16 if kind in ("first", "later") else F16)
            have = host(got[at]).reshape(want.shape)
            assert (np.abs(have - want) <= bound + np.expm1(moved) * spread).all(), (kind, b)


@pytest.mark.parametrize("n", [3, 70, 200])
def test_offsets_that_fall_touch_nothing_else(n):
    """Offsets in no order, negative ones and ones past the rows among them: calls end, pages of no table and memory around the
    cache stay as they were, and the next sound call is right."""
    from larder_amd import attention
    rng = np.random.default_rng(n)
    t, heads, width, page = 700, 2, 64, 32
    wide = random_cache(rng, 60, heads, width, page)
    before = [x.clone() for x in wide]
    cache = attention.KVCache(*(x[20:40] for x in wide))
    table = ints(rng.integers(0, 12, (n, 4)))          # pages 12 .. 19 of the cache are nobody's
    lens = ints(rng.integers(-3, 140, n))
    q, k, v = (normal(rng, t, h, width, dtype=F16) for h in (4, heads, heads))
    for _ in range(6):
        cu = rng.integers(-40, t + 100, n + 1)
        cu[rng.integers(0, n + 1)] = rng.choice([-2 ** 31, 2 ** 31 - 1])
        cu = ints(cu)
        outs = [*attention.append_rows(cache, q, k, v, table, lens, cu=cu, freq=frequencies(16), keys=True),
                *attention.read_rows(cache, table, cu, t, dtype=F16), attention.prompt_rows(q, k, v, cu),
                attention.prompt_rows(q, k, v, cu, cu_k=ints(rng.integers(-40, t + 100, n + 1))),
                attention.attend_rows(q, cache, table, lens, cu=cu), attention.attend_rows(q, cache, table, lens, cu=cu, longest=1)]
        assert all(o.shape[0] == t for o in outs)
        for a, b in zip(wide, before):
            a, b = (x.view(torch.uint8) for x in (a, b))
            assert torch.equal(a[:20], b[:20]) and torch.equal(a[32:], b[32:])
    cu = [0, 300, 300, 333]
    got = attention.prompt_rows(q[:333], k[:333], v[:333], ints(cu))
    check_prompt(got, q[:333], k[:333], v[:333], cu, cu, width ** -0.5, F16)


def test_attend_more_rows_than_a_grid_has_workgroups():
    """2^24 rows and heads and some: each is joined. One sequence of more rows than tokens, most of which see none."""
    from larder_amd import attention
    rng = np.random.default_rng(37)
    t, n = (1 << 19) + 1, 600
    cache = random_cache(rng, 19, 4, 64, 32)
    table = rng.permutation(19).astype(np.int32)[None]
    q = torch.ones(t, 32, 64, dtype=F16, device="cuda")
    q[-n:] = normal(rng, n, 32, 64, dtype=F16)
    torch.full((t * 32 * 64,), 7.0, dtype=F16, device="cuda")  # what the output is allocated from
    got = attention.attend_rows(q, cache, ints(table), ints([n]), cu=ints([0, t]))
    assert not got[:-n].any()
    check_attend(got[-n:], q[-n:], cache, table, [n], [0, n], 64 ** -0.5, F16)
