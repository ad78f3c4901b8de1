"""Host logic of the norms, the pages and the chunks over the cache: refusals, workspaces and what a launch covers, without a
GPU."""
import ctypes
import math
import random

import numpy as np
import pytest
import torch

from larder_amd import _lib, attention, pages, trunk

P = ctypes.c_void_p(16)  # never dereferenced: every call below is refused while its arguments are checked
ODD = ctypes.c_void_p(24)


def refused(L, code, word, name, *args):
    rc = getattr(L, name)(*args, None)
    assert rc == code and word in L.lmoe_error(), (rc, L.lmoe_error())


def test_norms_refuse(built_lib):
    L = built_lib

    def norm(x=P, dt=2, w=P, wdt=2, T=2, heads=1, H=64, eps=1e-6, out=P, group=0, scales=None):
        return x, dt, 64, 0, None, 0, 0, w, wdt, T, heads, H, eps, out, group, scales, None, 0, 0

    refused(L, _lib.EINVAL, b"dtype", "lmoe_norm_rows", *norm(dt=3))
    refused(L, _lib.EINVAL, b"dtype", "lmoe_norm_rows", *norm(wdt=1))
    refused(L, _lib.ESHAPE, b"channels", "lmoe_norm_rows", *norm(H=0))
    refused(L, _lib.ESHAPE, b"rows", "lmoe_norm_rows", *norm(T=-1))
    refused(L, _lib.ESHAPE, b"more than a launch", "lmoe_norm_rows", *norm(T=1 << 40))
    refused(L, _lib.ESHAPE, b"rows", "lmoe_norm_rows", *norm(T=1 << 62, heads=4))
    for eps in (0.0, -1.0, float("inf"), float("nan")):
        refused(L, _lib.EINVAL, b"eps", "lmoe_norm_rows", *norm(eps=eps))
    for group in (-1, 16, 48, 128):
        refused(L, _lib.ESHAPE, b"scales", "lmoe_norm_rows", *norm(group=group, scales=P))
    refused(L, _lib.EINVAL, b"null", "lmoe_norm_rows", *norm(group=32))
    refused(L, _lib.EINVAL, b"null", "lmoe_norm_rows", *norm(w=None))
    assert L.lmoe_norm_rows(*norm(T=0, x=None), None) == 0
    refused(L, _lib.EINVAL, b"dtype", "lmoe_read_codes", P, P, 64, 32, P, 5)
    refused(L, _lib.ESHAPE, b"groups", "lmoe_read_codes", P, P, 65, 32, P, 0)
    refused(L, _lib.ESHAPE, b"groups", "lmoe_read_codes", P, P, 64, 0, P, 0)
    refused(L, _lib.EINVAL, b"null", "lmoe_read_codes", P, None, 64, 32, P, 0)
    refused(L, _lib.EALIGN, b"aligned", "lmoe_read_codes", ODD, P, 64, 32, P, 0)
    assert L.lmoe_read_codes(None, None, 0, 32, None, 0, None) == 0


def test_pages_refuse(built_lib):
    L = built_lib

    def take(refs=P, n=4, table=P, B=2, width=3, lens=P, page=64, src=P, ws=P, wsb=1 << 20):
        return refs, n, table, B, width, lens, None, page, src, P, P, ws, wsb

    for bad in (0, -1, 2 ** 31 - 1):
        refused(L, _lib.ESHAPE, b"pages", "lmoe_pages_take", *take(n=bad))
    refused(L, _lib.ESHAPE, b"tokens", "lmoe_pages_take", *take(page=48))
    refused(L, _lib.ESHAPE, b"places", "lmoe_pages_take", *take(width=0))
    refused(L, _lib.ESHAPE, b"int", "lmoe_pages_take", *take(width=2 ** 31 // 64))
    refused(L, _lib.ESHAPE, b"int", "lmoe_pages_take", *take(width=1 << 20, B=1 << 12))
    refused(L, _lib.EINVAL, b"null", "lmoe_pages_take", *take(lens=None))
    refused(L, _lib.EWORKSPACE, b"workspace", "lmoe_pages_take", *take(ws=None))
    refused(L, _lib.EWORKSPACE, b"workspace", "lmoe_pages_take", *take(wsb=8))
    assert L.lmoe_pages_take(*take(B=0, refs=None), None) == 0
    # where tasks begin, their ranks, the pages that are given, the counts of a large pool's stretches
    assert L.lmoe_pages_take_workspace_bytes(2, 3, 4) == 4 * (2 + 6 + 4 + 1)
    assert L.lmoe_pages_take_workspace_bytes(64, 2048, 100000) == 4 * (64 + 64 * 2048 + 100000 + 13)
    assert L.lmoe_pages_take_workspace_bytes(0, 3, 4) == 0
    refused(L, _lib.ESHAPE, b"tokens", "lmoe_pages_free", P, 4, P, 2, 3, P, 100)
    refused(L, _lib.ESHAPE, b"more than a launch", "lmoe_pages_free", P, 4, P, 1 << 20, 1 << 20, P, 64)
    refused(L, _lib.EINVAL, b"null", "lmoe_pages_free", P, 4, P, 2, 3, None, 64)
    refused(L, _lib.ESHAPE, b"sequences", "lmoe_pages_fork", P, 4, P, 2, 3, P, -1, P)
    refused(L, _lib.EINVAL, b"null", "lmoe_pages_fork", P, 4, P, 2, 3, None, 2, P)
    refused(L, _lib.EINVAL, b"null", "lmoe_pages_compact", P, 4, P, P, None, P, P, 64)
    refused(L, _lib.EWORKSPACE, b"workspace", "lmoe_pages_compact", P, 4, P, P, P, P, P, 4)
    assert L.lmoe_pages_compact_workspace_bytes(8192) == 8 and L.lmoe_pages_compact_workspace_bytes(8193) == 12
    refused(L, _lib.EINVAL, b"null", "lmoe_pages_renumber", P, 2, 3, 4, None, P)

    def copy(k=P, n=4, page=64, heads=1, D=64, pairs=2, src=P):
        return k, P, P, P, n, page, heads, D, src, P, pairs

    refused(L, _lib.ESHAPE, b"channels", "lmoe_pages_copy", *copy(D=96))
    refused(L, _lib.ESHAPE, b"tokens", "lmoe_pages_copy", *copy(page=16))
    refused(L, _lib.ESHAPE, b"copies", "lmoe_pages_copy", *copy(pairs=-1))
    refused(L, _lib.EINVAL, b"null", "lmoe_pages_copy", *copy(src=None))
    refused(L, _lib.EALIGN, b"aligned", "lmoe_pages_copy", *copy(k=ODD))
    assert L.lmoe_pages_copy(*copy(pairs=0, k=None), None) == 0


def test_chunks_refuse(built_lib):
    L = built_lib

    def chunk(q=P, dt=1, st=64, T=2, qh=2, h=1, D=64, cu=P, B=1, width=1, pages=1, page=64, longest=64, scale=0.1, ws=P, wsb=1 << 30):
        return q, dt, st, 64, T, qh, h, D, cu, P, B, P, width, P, P, P, P, pages, page, longest, scale, ws, wsb, P

    refused(L, _lib.EINVAL, b"dtype", "lmoe_kv_chunk", *chunk(dt=0))
    refused(L, _lib.ESHAPE, b"channels", "lmoe_kv_chunk", *chunk(D=96))
    refused(L, _lib.ESHAPE, b"tokens", "lmoe_kv_chunk", *chunk(page=16))
    refused(L, _lib.ESHAPE, b"query heads", "lmoe_kv_chunk", *chunk(qh=3, h=2))
    refused(L, _lib.ESHAPE, b"places", "lmoe_kv_chunk", *chunk(width=2 ** 31 // 64))
    refused(L, _lib.ESHAPE, b"rows", "lmoe_kv_chunk", *chunk(longest=0))
    refused(L, _lib.ESHAPE, b"sequence", "lmoe_kv_chunk", *chunk(B=0))
    refused(L, _lib.ESHAPE, b"offsets", "lmoe_kv_chunk", *chunk(cu=None))
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        refused(L, _lib.EINVAL, b"scale", "lmoe_kv_chunk", *chunk(scale=scale))
    refused(L, _lib.EINVAL, b"null", "lmoe_kv_chunk", *chunk(q=None))
    refused(L, _lib.EALIGN, b"aligned", "lmoe_kv_chunk", *chunk(q=ODD))
    refused(L, _lib.EALIGN, b"aligned", "lmoe_kv_chunk", *chunk(st=65))
    refused(L, _lib.ESHAPE, b"pages of", "lmoe_kv_chunk", *chunk(h=1 << 20, qh=1 << 20, D=256, page=128))
    refused(L, _lib.ESHAPE, b"rows of", "lmoe_kv_chunk", *chunk(T=1 << 30, qh=8))
    refused(L, _lib.ESHAPE, b"more than a launch", "lmoe_kv_chunk", *chunk(T=1 << 26, qh=512, h=512))
    refused(L, _lib.EWORKSPACE, b"workspace", "lmoe_kv_chunk", *chunk(longest=100000, width=2000, wsb=16))
    refused(L, _lib.EWORKSPACE, b"workspace", "lmoe_kv_chunk", *chunk(longest=100000, width=2000, ws=None))
    assert L.lmoe_kv_chunk(*chunk(T=0), None) == 0


def test_chunk_workspace(built_lib):
    """Two places for each workgroup's pairs: width sums, a maximum and a weight; where each row and head has its own. A long history
    under few rows is split, many rows are not, and the largest sizes stay in bounds."""
    f = built_lib.lmoe_kv_chunk_workspace_bytes
    for t, q, h, d, b, n in ((48, 32, 4, 128, 1, 131048), (17, 4, 4, 64, 3, 2 ** 31 - 1), (100, 16, 2, 256, 5, 9000)):
        groups, rest = divmod(f(t, q, h, d, b, n) - t * q * 8, 2 * 128 * (d + 4) * 4)
        assert rest == 0 and groups % h == 0 and h < groups <= (256 if d == 256 else 512)
    assert f(8192, 32, 4, 128, 1, 8192) == 0 and f(48, 32, 4, 128, 1, 60) == 0
    assert f(0, 4, 4, 64, 1, 100) == 0 and f(4, 3, 2, 64, 1, 100) == 0 and f(4, 4, 4, 64, 0, 100) == 0


@pytest.mark.parametrize("longest", [-1, 0, 5, 2 ** 31, 2 ** 32, 10 ** 30])
def test_any_longest_sizes_a_launch(monkeypatch, built_lib, longest):
    sizes = []
    monkeypatch.setattr(attention, "_device", lambda *a: 0)
    monkeypatch.setattr(attention, "_launch", lambda dev, name, *args: sizes.append(args))
    cache, i = attention.KVCache.empty(1, 1, 64, device="cpu"), torch.tensor([0, 3], dtype=torch.int32)
    attention.chunk_rows(torch.zeros(3, 2, 64, dtype=torch.float16), cache, torch.zeros(1, 20, dtype=torch.int32), i[1:], cu=i, longest=longest)
    assert sizes[0][19] == min(max(longest, 1), 20 * 64)
    assert sizes[0][22] == built_lib.lmoe_kv_chunk_workspace_bytes(3, 2, 1, 64, 1, sizes[0][19])


@pytest.mark.parametrize("rows", [128, 256])
def test_every_tile_of_pairs_has_a_workgroup(rows):
    """nth_chunk_tile's numbering, restated: T group / rows + B tiles (one sequence: as many as it has) hold every sequence's, by
    either of its two ways; without offsets too."""
    rng = random.Random(rows)
    for turn in range(300):
        group, n = rng.choice([1, 2, 3, 7, 8, 40, 200]), rng.choice([1, 2, 5, 64, 65, 130])
        counts = [1] * n if turn % 5 == 0 else [rng.choice([0, 1, 3, 17, 128, 129, 1000]) for _ in range(n)]
        T, cu = sum(counts), np.cumsum([0] + counts)
        if not T:
            continue
        tiles = -(-T * group // rows) if n == 1 else T * group // rows + n
        have = [-(-c * group // rows) for c in counts]
        for end in (0, n - 1):
            have[end] = max(have[end], 1)
        assert sum(have) <= tiles
        begin = [int(cu[b]) * group // rows + b for b in range(n)]
        if n > 64:
            seen = set()
            for nth in range(tiles):
                turned = (nth & ~7) | ((nth + (nth >> 3)) & 7) if nth < (tiles & ~7) else nth
                task = tiles - 1 - turned
                b = max(i for i in range(n) if begin[i] <= task)
                if turn % 5 == 0:  # the closed form that stands for the search
                    guess = min(n - 1, task * rows // (group + rows) + 1)
                    while begin[guess] > task:
                        guess -= 1
                    assert guess == b
                seen.add((b, task - begin[b]))
            assert all((b, t) in seen for b in range(n) for t in range(have[b]))


def test_tensors_off_the_gpu_are_refused():
    x, i = torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32)
    cache = attention.KVCache.empty(2, 1, 64, device="cpu")
    for call in (lambda: trunk.norm_rows(x, x[0]), lambda: trunk.read_codes(x.to(torch.float8_e4m3fn), torch.zeros(2, 1)),
                 lambda: pages.take_pages(i, i[:, None], i), lambda: pages.free_pages(i, i[:, None], i),
                 lambda: pages.fork_pages(i, i[:, None], i), lambda: pages.compact_pages(i, i[:, None]),
                 lambda: pages.copy_pages(cache, i, i),
                 lambda: attention.chunk_rows(torch.zeros(2, 1, 64, dtype=torch.float16), cache, i[:, None], i)):
        with pytest.raises(ValueError, match="GPU"):
            call()


def test_the_trunks_attention_in_chunks_refuses_before_it_writes(monkeypatch):
    def affine(n, k):
        return torch.zeros(n, k // 8, dtype=torch.int32), *(torch.zeros(n, k // 64, dtype=torch.bfloat16) for _ in range(2)), 64
    written = []
    monkeypatch.setattr(trunk, "qmv_rows", lambda x, w, *_: torch.zeros(x.shape[0], w.shape[0], dtype=torch.bfloat16))
    monkeypatch.setattr(attention, "append_rows", lambda *a, **_: written.append(a) or (a[1], a[2]))
    cu, w = torch.tensor([0, 2], dtype=torch.int32), torch.zeros(64, dtype=torch.bfloat16)
    args = dict(qkv=affine(8 * 64, 128), out=affine(128, 4 * 64), cache=attention.KVCache.empty(1, 2, 64, device="cpu"),
                table=torch.zeros(1, 1, dtype=torch.int32), lens=cu[1:], cu=cu)
    for kw, why in ((dict(prompt="chunk", cu=None), "offsets"), (dict(prompt="chunks"), "chunk"), (dict(norms=(w[:63], w, 1e-6)), "weight"),
                    (dict(norms=(w, w.half(), 1e-6)), "weight|GPU"), (dict(norms=(w, w, 0.0)), "eps")):
        with pytest.raises(ValueError, match=why):
            trunk.attention_rows(torch.zeros(2, 128, dtype=torch.bfloat16), **{**args, **kw})
    assert not written


@pytest.mark.parametrize("rows", [128, 256])
def test_stretches_hold_every_key_once(rows):
    """TileLine's two ways of cutting a head's tiles, restated: stretches one behind another hold every tile's keys once, in order,
    none but a tile's first piece without keys, and two stretches never begin inside a tile at the same key."""
    rng = random.Random(rows + 1)
    start = 192 if rows == 128 else 320
    for turn in range(400):
        group, n, room = rng.choice([1, 2, 3, 7, 8, 40, 200]), rng.choice([1, 1, 2, 5, 64, 70]), rng.choice([64, 640, 10 ** 9])
        counts = [rng.choice([0, 1, 3, 17, 128, 700]) for _ in range(n)]
        lens = [rng.choice([0, 1, c // 2, c, c + 63, c + 64, c + 1000, c + 30000]) for c in counts]
        tiles = [-(-c * group // rows) for c in counts]

        def seen(b, t):
            return min(lens[b] - counts[b] + (min(t * rows + rows, counts[b] * group) - 1) // group + 1, room)

        def cost(b, t):
            return t * (group * (max(lens[b] - counts[b], 0) + start) + rows / 2 * (t + 1))

        want = [(b, t) for b in range(n) for t in range(tiles[b])]
        total = sum(cost(b, tiles[b]) for b in range(n))
        of = rng.choice([2, 3, 16, 60, 128, 512])

        def place(x):
            for b in range(n):
                if x < cost(b, tiles[b]):
                    t = max(t for t in range(tiles[b]) if cost(b, t) <= x)
                    key = int(max((x - cost(b, t)) / group - start, 0.0)) & -64
                    return (b, t + 1, 0) if key and seen(b, t) - key < 64 else (b, t, key)
                x -= cost(b, tiles[b])
            return (n, 0, 0)

        each = total / of
        if each / group < 128:
            of = max(int(total / group / 128), 1)
            each = total / of
        ends = [place(math.floor(each * i)) for i in range(of)] + [(n, 0, 0)]
        ways = [list(zip(ends, ends[1:]))]
        if n == 1 and tiles[0]:
            per = rng.choice([2, 3, 8, 42])
            cut = []
            for one in range(tiles[0] * per):
                t, i = divmod(one, per)
                step = ((max(seen(0, t), 1) - 1) // (per * 64) + 1) * 64
                if i == 0 or i < -(-seen(0, t) // step):
                    cut.append(((0, t, i * step), (0, t, (i + 1) * step) if (i + 1) * step < seen(0, t) else (0, t + 1, 0)))
            ways.append(cut)
        for stretches in ways:
            held = []
            for (b, t, key), end in stretches:
                while b < n and (b, t, key) < end:
                    if t >= tiles[b]:
                        b, t, key = b + 1, 0, 0
                        continue
                    stop = min(seen(b, t), end[2]) if end[:2] == (b, t) else seen(b, t)
                    assert key == 0 or stop > key
                    held.append((b, t, key, stop))
                    t, key = t + 1, 0
            assert [x[:2] for x in held if x[2] == 0] == want
            for a, z in zip(held, held[1:] + [(n, 0, 0, 0)]):
                assert z[2] == a[3] and z[:2] == a[:2] if z[2] else a[3] == seen(*a[:2])
