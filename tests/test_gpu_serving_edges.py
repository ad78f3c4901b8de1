"""GPU parity at the ends of what the norms, the pages and the chunks over the cache take, against float64 and the oracles.

Tolerances: those of test_gpu_chunk.py and test_gpu_norm.py, or equality."""
import random

import numpy as np
import pytest
import torch

from oracle import pages as pool_ref
from test_gpu_attention import BF16, F16, ints, normal, page_table, poisoned_memory, random_cache  # noqa: F401
from test_gpu_chunk import check, check_long
from test_gpu_norm import check as check_norm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("longest", [None, 64])
@pytest.mark.parametrize("heads,width", [(2, 64), (1, 128), (1, 256)])
@pytest.mark.parametrize("apart", [7, 15, 16, 19, 22])
def test_chunk_float16_pages_far_apart(apart, heads, width, longest):
    """Values of two pages of one tile, the larger scale 2^apart times the other: rows that see the smaller page alone, or give all of
    their weight to it, have its values to the last bit. (Rows of both stay finite: the larger page's codes are 1 at most, and the
    smaller one's scale is 2^7 or less: 448 2^7 < 65504.)"""
    from larder_amd import attention
    rng = np.random.default_rng(apart)
    cache = random_cache(rng, 4, heads, width, 32)
    codes = rng.choice([1, 2, 5, 0x2d, 0x33, 0x38, 0x39, 0x3d, 0x41, 0x59, 0x7e], (4, heads, 32, width)) | rng.integers(0, 2, (4, heads, 32, width)) << 7
    codes[2:] = rng.integers(0, 0x39, (2, heads, 32, width))
    cache.v.view(torch.uint8).copy_(torch.from_numpy(codes.astype(np.uint8)))
    cache.v_scale[:2], cache.v_scale[2:] = 2.0 ** (14 - apart), 2.0 ** 14
    # (a sequence whose smaller page comes first; one whose larger page comes first, with keys that no row gives any weight to)
    table, lens, cu = np.array([[0, 2], [3, 1]]), [64, 60], [0, 64, 90]
    cache.k_scale.fill_(2.0 ** -6)
    cache.k.view(torch.uint8)[3] = 0xf8  # -256
    cache.k.view(torch.uint8)[1] &= 0x3f
    q = normal(rng, 90, 3 * heads, width, dtype=F16)
    q[64:] = 16.0
    got = attention.chunk_rows(q, cache, ints(table), ints(lens), ints(cu), longest=longest)
    check(got, q, cache, table, lens, cu, width ** -0.5, F16)
    # a row of one token is that token, and each of a page's first rows lies within the page's own values
    first = cache.v[0, :, 0].float() * cache.v_scale[0, 0]
    assert torch.equal(got[0].view(heads, 3, width), first[:, None].expand(heads, 3, width).to(F16))
    alone = attention.chunk_rows(q[:32], cache, ints(table[:1, :1]), ints([32]), ints([0, 32]), longest=64)
    assert (got[:32].double() - alone.double()).abs().max() <= 2.0 ** -10 * alone.double().abs().max()


@pytest.mark.parametrize("sequences,shared,free", [(2, 1, 0), (3, 1, 1), (40, 7, 0), (40, 7, 11), (700, 100, 300), (3000, 900, 40),
                                                   (2500, 1, 2300)])
def test_take_where_pages_run_out(sequences, shared, free):
    """Groups of sequences that share their last page and all or some of whom write to it, with fewer free pages than writers."""
    from larder_amd import pages as own
    rng = random.Random(sequences + free)
    page, pages = 32, shared + free
    for writes in (1.0, 0.8, 0.5):
        table = [[rng.randrange(shared), -1, -1] for _ in range(sequences)]
        refs = [0] * pages
        for row in table:
            refs[row[0]] += 1
        order = list(range(pages))
        rng.shuffle(order)
        table = [[order[p] if p >= 0 else -1 for p in row] for row in table]
        refs = [r for _, r in sorted(zip(order, refs))]
        refs = [r if r or p not in order[:shared] else 9 for p, r in enumerate(refs)]  # (a page that others hold)
        rows = [rng.choice([1, 3, 40, 64]) if rng.random() < writes else 0 for _ in range(sequences)]
        lens, cu = [7 + r for r in rows], [int(x) for x in np.cumsum([0] + rows)]
        want = pool_ref.take(refs, table, lens, cu, page)
        for _ in range(3):
            r, t = ints(refs), ints(table)
            got = own.take_pages(r, t, ints(lens), ints(cu), page=page)
            for a, b in zip((r, t, *got), want):
                assert a.tolist() == b


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_chunk_of_a_table_with_room_for_2_31_tokens(dtype):
    """The last 32-token page of the longest table there is: its tokens are seen, and a NaN in the very last by the last row alone."""
    from larder_amd import attention
    rng = np.random.default_rng(31)
    places = (2 ** 31 - 1) // 32
    cache = random_cache(rng, 2, 1, 64, 32)
    cache.k_scale.fill_(1.0), cache.v_scale.fill_(0.5)
    cache.k.view(torch.uint8)[0] = 0xc0  # -2: scores of -128 against the last page's 128
    cache.k.view(torch.uint8)[1] = 0x40
    cache.v.view(torch.uint8)[1, 0, 31, 5] = 0x7f
    table = torch.zeros((1, places), dtype=torch.int32, device="cuda")
    table[0, -1] = 1
    q = torch.ones(2, 3, 64, dtype=dtype, device="cuda")
    got = attention.chunk_rows(q, cache, table, ints([32 * places]), ints([0, 2]), scale=1.0).double()
    v = cache.v[1, 0].double() * 0.5
    for row, n in ((0, 31), (1, 32)):
        want, spread = v[:n].mean(0), v[:n].abs().mean(0)
        off = (got[row] - want).abs()
        # (equal weights, sums of 32 values at most: the result's rounding and a few of float32; float16 has steps of 2^-24)
        ok = off <= torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -18 * spread + 2.0 ** -25
        assert (ok | torch.isnan(want)).all(), (row, off.max())
        assert torch.isnan(got[row]).any(0).tolist() == [n == 32 and c == 5 for c in range(64)]


@pytest.mark.parametrize("h", [8, 500, 512, 2000, 16400])
def test_norm_of_small_channels_beside_large_ones(h):
    """Rows whose squares pass float32: channels 2^-120 of the largest keep their bits, and eps counts where it is as large."""
    rng = torch.Generator(device="cuda").manual_seed(h)
    x = torch.randn((7, h), generator=rng, device="cuda") * 2.0 ** 66
    x[1:4, ::2] *= 2.0 ** -110
    x[4, 1::3] *= 2.0 ** -120
    x[5] *= 2.0 ** 58
    w = 1 + torch.rand(h, generator=rng, device="cuda")
    check_norm(x, None, w, 1e-6)
    check_norm(x, x.flip(1), w, 1e38)
    check_norm(x, None, w, 3e38)
    check_norm(x, None, w, 1e38, group=h)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("q_heads,heads,width", [(32, 8, 64), (32, 8, 128), (16, 8, 256)])
@pytest.mark.parametrize("sequences", [2, 5, 12, 40, 64])
def test_chunk_whole_tiles_of_many_sequences(dtype, q_heads, heads, width, sequences):
    """More workgroups than places, each a whole tile, the longest tiles first: sequences of few and many rows over no and long
    histories, the first, the last and one between without rows; rows before and behind them."""
    from larder_amd import attention
    rng = np.random.default_rng(100 * sequences + width)
    parts = rng.random(sequences) ** 2
    if sequences > 3:
        parts[[0, sequences // 2, -1]] = 0
    rows = [int(x) for x in np.floor(2600 * parts / parts.sum())]
    past = [int(rng.choice([0, 1, 255, 256, 700, 1300])) for _ in rows]
    lens = [r + p for r, p in zip(rows, past)]
    if sequences > 3:
        lens[1] = rows[1] // 2  # more rows than tokens
    cu = [5] + [5 + int(x) for x in np.cumsum(rows)]
    t, long = cu[-1] + 3, max(lens)
    assert attention._chunk_workspace(t, q_heads, heads, width, sequences, long) == 0
    assert (t * q_heads // heads // (256 if width == 128 else 128) + 1) * heads > (512 if width == 64 else 256)
    table, n = page_table(rng, [-(-x // 64) for x in lens])
    cache = random_cache(rng, n, heads, width, 64)
    q = normal(rng, t, q_heads, width, dtype=dtype)
    got = attention.chunk_rows(q, cache, ints(table), ints(lens), ints(cu), longest=long)
    assert (got[:5] == 0).all() and (got[cu[-1]:] == 0).all() and not torch.isnan(got).any()
    check_long(got, q, cache, table, lens, cu, width ** -0.5, dtype, some=[0, q_heads // 2 - 1, q_heads - 1])


@pytest.mark.parametrize("lens", [[2 ** 31 - 1, 300], [70, 2 ** 31 - 100], [2 ** 31 - 320, 2 ** 31 - 1]])
def test_chunk_of_lengths_at_an_ints_end(lens):
    """Sequences of far more tokens than their table has places: every row sees all the table's, the others what they see."""
    from larder_amd import attention
    rng = np.random.default_rng(lens[0] % 97)
    rows, cu, page, places = [40, 30], [0, 40, 70], 64, 400
    table, n = page_table(rng, [places, places])
    cache = random_cache(rng, n, 2, 128, page)
    q = normal(rng, 70, 8, 128)
    assert attention._chunk_workspace(70, 8, 2, 128, 2, places * page)
    got = attention.chunk_rows(q, cache, ints(table), ints(lens), ints(cu))
    # (all of the table, for a row each: the same sums with no length beyond it)
    for b in range(2):
        for r in (0, rows[b] - 1):
            sees = min(lens[b] - rows[b] + r + 1, places * page)
            one = q[cu[b] + r][None]
            check_long(got[cu[b] + r][None], one, cache, table[b][None], [sees], [0, 1], 128 ** -0.5, BF16)
    assert not torch.isnan(got).any()


@pytest.mark.parametrize("q_heads,heads,width,rows", [(3, 1, 64, 100), (8, 2, 128, 90), (16, 1, 128, 700), (4, 2, 256, 60)])
@pytest.mark.parametrize("fill", [-1, 0, 3, 129, 0x7fffffff, -2 ** 31])
def test_chunk_writes_its_rows_alone(q_heads, heads, width, rows, fill):
    """Right and wild offsets, lengths and tables; a workspace that holds small and large whole numbers beforehand: what lies around
    the output and the workspace keeps its value."""
    from larder_amd import _lib, attention
    rng, pick = np.random.default_rng(width + rows), random.Random(rows)
    page, room, around = 32, 300, 4096
    cache = random_cache(rng, 40, heads, width, page)
    q = normal(rng, rows, q_heads, width)
    codes = [t.data_ptr() for t in cache]
    wild = [-2 ** 31, -5, -1, 0, 1, 7, rows // 2, rows, 1000, 9600, 2 ** 31 - 1]
    split = 0
    for n in (1, 3, 65):
        for turn in range(3):
            if turn == 0:  # right ones, rows of no sequence at both ends
                cu = sorted(rng.integers(1, rows, n + 1).tolist())
                lens, table = [9000 + 7 * b for b in range(n)], rng.integers(0, 40, (n, room)).tolist()
            else:
                cu, lens = [pick.choice(wild) for _ in range(n + 1)], [pick.choice(wild) for _ in range(n)]
                table = [[pick.choice(wild) for _ in range(room)] for _ in range(n)]
            need = attention._chunk_workspace(rows, q_heads, heads, width, n, room * page)
            split += need > 0
            ws = torch.full((need // 4 + 2 * around,), fill, dtype=torch.int32, device="cuda")
            out = torch.full((rows * q_heads * width // 2 + 2 * around,), 77, dtype=torch.int32, device="cuda")
            cu_t, lens_t, table_t = ints(cu), ints(lens), ints(table)
            print("writes", q_heads, width, fill, n, turn, flush=True)
            _lib.call("lmoe_kv_chunk", q.data_ptr(), _lib.BF16, q_heads * width, width, rows, q_heads, heads, width, cu_t.data_ptr(),
                      lens_t.data_ptr(), n, table_t.data_ptr(), room, codes[0], codes[1], codes[2], codes[3], 40, page, room * page,
                      0.1, ws.data_ptr() + 4 * around, need, out.data_ptr() + 4 * around, _lib.stream())
            torch.cuda.synchronize()
            for t, x, inside in ((ws, fill, need // 4), (out, 77, rows * q_heads * width // 2)):
                assert t[:around].eq(x).all() and t[around + inside:].eq(x).all(), (n, turn)
            if turn == 0:
                got = out[around:around + rows * q_heads * width // 2].view(torch.bfloat16).view(rows, q_heads, width)
                assert torch.equal(got, attention.chunk_rows(q, cache, table_t, lens_t, cu_t, scale=0.1))
    assert split


@pytest.mark.parametrize("h", [8, 512, 2000, 16400])
@pytest.mark.parametrize("power", [-120, -60, 60, 110, 120])
def test_norm_of_large_rows_with_weights_of_all_sizes(h, power):
    """Rows whose squares pass float32, with weights down to 2^-120 and up to 2^120: results that float32 holds are right."""
    rng = torch.Generator(device="cuda").manual_seed(h)
    x = torch.randn((5, h), generator=rng, device="cuda").clamp(-4, 4) * 2.0 ** 70
    x[1:3, ::2] *= 2.0 ** -100
    x[3] *= 2.0 ** 50
    w = (1 + torch.rand(h, generator=rng, device="cuda")) * 2.0 ** power
    check_norm(x, None, w, 1e-6)
