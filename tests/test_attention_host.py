"""The host side of the trunk's attention without a GPU: rotary frequencies, the entry points' refusals, their workspace, and
how a call's pages are dealt to workgroups."""
import ctypes
import math

import numpy as np
import pytest
import torch

from larder_amd import _lib, attention


def test_rotary_freq():
    f, gain = attention.rotary_freq(8, 10000.0, device="cpu")
    assert torch.equal(f, 10000.0 ** (-torch.arange(4, dtype=torch.float64) / 4)) and gain == 1.0
    g, _ = attention.rotary_freq(8, 10000.0, "linear", 4.0, device="cpu")
    assert torch.equal(g, f / 4)
    g, _ = attention.rotary_freq(8, 10000.0, "ntk", 4.0, device="cpu")
    assert g[0] == 1.0 and math.isclose(float(g[-1]), float(f[-1]) / 4, rel_tol=1e-12)  # the slowest interpolated
    f, _ = attention.rotary_freq(128, 10000.0, device="cpu")
    g, gain = attention.rotary_freq(128, 10000.0, "yarn", 8.0, 4096, device="cpu")
    assert math.isclose(gain, 0.1 * math.log(8) + 1)
    turns = 4096 * f / (2 * math.pi)
    assert torch.allclose(g[turns > 40], f[turns > 40]) and torch.allclose(g[turns < 0.8], f[turns < 0.8] / 8)
    assert ((g <= f) & (g >= f / 8)).all() and (torch.diff(g) < 0).all()
    # factor 1: f keep + f (1 - keep), three roundings of 2^-53
    assert torch.allclose(attention.rotary_freq(128, 10000.0, "yarn", 1.0, 4096, device="cpu")[0], f, rtol=2.0 ** -51, atol=0)


@pytest.mark.parametrize("width,original,low,high", [(128, 131072, 45, 70), (128, 65536, 40, 65), (128, 4096, 20, 46),
                                                     (64, 10 ** 7, 37, 50), (64, 10 ** 9, 53, 63), (32, 10 ** 9, 26, 31)])
def test_yarn_ramps_end_where_the_published_ones_do(width, original, low, high):
    """Base 10,000: the pair that turns n times in `original` positions is width ln(original / (2 pi n)) / (2 ln 10,000), 32
    turns of it rounded down and one turn rounded up, within [0, width - 1]: also where that lies past the last pair."""
    turns = [width * math.log(original / (2 * math.pi * n)) / (2 * math.log(10000)) for n in (32, 1)]
    assert (max(math.floor(turns[0]), 0), min(math.ceil(turns[1]), width - 1)) == (low, high)
    got, _ = attention.rotary_freq(width, 10000.0, "yarn", 8.0, original, device="cpu")
    for i, f in enumerate(got.tolist()):
        keep = 1 - min(max((i - low) / (high - low), 0), 1)
        assert math.isclose(f, 10000 ** (-2 * i / width) * (keep + (1 - keep) / 8), rel_tol=1e-12)


@pytest.mark.parametrize("kw", [dict(width=7), dict(width=0), dict(width=8, factor=0.5), dict(width=8, kind="yarn"),
                                dict(width=8, kind="other")])
def test_rotary_freq_refuses(kw):
    with pytest.raises(ValueError):
        attention.rotary_freq(**kw, device="cpu")


def test_tensors_off_the_gpu_are_refused():
    x, i = torch.zeros(1, 1, 64, dtype=torch.float16), torch.zeros(1, dtype=torch.int32)
    cache = attention.KVCache.empty(1, 1, 64, device="cpu")
    freq = torch.zeros(32, dtype=torch.float64)
    cu = torch.tensor([0, 1], dtype=torch.int32)
    for call in (lambda: attention.rope_rows(x, i, freq), lambda: attention.append_rows(cache, x, x, x, i[None], i),
                 lambda: attention.attend_rows(x, cache, i[None], i), lambda: attention.read_rows(cache, i[None], cu, 1),
                 lambda: attention.prompt_rows(x, x, x, cu)):
        with pytest.raises(ValueError, match="GPU"):
            call()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_rows_of_any_layout_have_strides_the_kernels_read(dtype):
    """Aligned strides, and the same values through them: also where an axis of size one has a stride of its own, which torch
    calls contiguous whatever it is."""
    step = 16 // torch.zeros((), dtype=dtype).element_size()
    wide = torch.arange(9 * 1027, dtype=torch.float32).remainder(97).to(dtype).view(9, 1027)
    cols = torch.arange(9 * 3 * 129, dtype=torch.float32).remainder(89).to(dtype).view(9, 3, 129)
    rows = wide[:, :512].view(9, 4, 128)
    for x in (rows, rows[0:1], rows[3:4], rows[2:2], cols[:, 1:2, :128], cols[4:5, 2:3, 1:], cols[:, :, :128], rows[:, :, 1:65],
              rows[3:4, :1, ::2], wide[:, :1024].view(9, 8, 128), wide[:, :1024].view(9, 8, 128).transpose(0, 1), rows[:1].expand(5, 4, 128)):
        y, s0, s1 = attention._rows("f", "x", x)
        assert y.shape == x.shape and s0 % step == 0 and s1 % step == 0 and y.data_ptr() % 16 == 0
        if x.numel():
            assert torch.equal(torch.as_strided(y, y.shape, (s0, s1, 1), y.storage_offset()), x)


def test_keys_too_far_apart_for_the_prompt_kernel_are_copied():
    apart = attention._KEYS_APART
    wide = torch.zeros(3, apart, dtype=torch.float16)
    for n, copied in ((apart, True), (apart - 8, False)):
        x = wide.view(-1)[:3 * n].view(3, n)[:, 64:192].view(3, 2, 64)
        x.copy_(torch.arange(3 * 128).view(3, 2, 64))
        y, s0, s1 = attention._rows("f", "k", x, apart=apart)
        assert (s0, s1) == ((128, 64) if copied else (n, 64)) and torch.equal(y, x)
        assert attention._rows("f", "k", x[1:2], apart=apart)[1:] == (128, 64)


def affine(n, k):
    return torch.zeros(n, k // 8, dtype=torch.int32), *(torch.zeros(n, k // 64, dtype=torch.bfloat16) for _ in range(2)), 64


CU = torch.tensor([0, 2], dtype=torch.int32)


@pytest.mark.parametrize("kw,why", [
    (dict(prompt=True), "offsets"), (dict(prompt=(CU, 2)), "offsets"), (dict(prompt=(CU.long(), 2), cu=CU), "cu_k"),
    (dict(prompt=(CU[:1], 2), cu=CU), "cu_k"), (dict(prompt=(CU, -1), cu=CU), "total"), (dict(qkv=affine(7 * 64, 128)), "heads"),
    (dict(qkv=affine(4 * 64, 128)), "heads"), (dict(qkv=affine(8 * 64 + 8, 128)), "heads"), (dict(out=affine(128, 3 * 64)), "out"),
    (dict(out=affine(128, 4 * 64)[:2] + (None, 64)), "out")])
def test_the_trunks_attention_refuses_before_it_writes(monkeypatch, kw, why):
    """attention_rows on two key heads of 64: what one of its steps would refuse is refused before the cache is written."""
    from larder_amd import trunk
    written = []
    monkeypatch.setattr(trunk, "qmv_rows", lambda x, w, *_: torch.zeros(x.shape[0], w.shape[0], dtype=torch.bfloat16))
    monkeypatch.setattr(attention, "append_rows", lambda *a, **_: written.append(a) or (a[1], a[2]))
    args = dict(qkv=affine(8 * 64, 128), out=affine(128, 4 * 64), cache=attention.KVCache.empty(1, 2, 64, device="cpu"),
                table=torch.zeros(1, 1, dtype=torch.int32), lens=torch.tensor([2], dtype=torch.int32))
    with pytest.raises(ValueError, match=why):
        trunk.attention_rows(torch.zeros(2, 128, dtype=torch.bfloat16), **{**args, **kw})
    assert not written


@pytest.mark.parametrize("prompt", [None, True, "later"])
def test_the_trunks_attention_of_no_rows(monkeypatch, prompt):
    from larder_amd import trunk
    monkeypatch.setattr(trunk, "qmv_rows", lambda x, w, *_: torch.zeros(x.shape[0], w.shape[0], dtype=torch.bfloat16))
    monkeypatch.setattr(attention, "append_rows", lambda c, q, k, v, *a, **_: (q, k))
    monkeypatch.setattr(attention, "read_rows", lambda c, t, cu, n, **_: [torch.zeros(n, 2, 64, dtype=torch.bfloat16)] * 2)
    for f in ("attend_rows", "prompt_rows"):
        monkeypatch.setattr(attention, f, lambda q, *a, **_: q)
    cu = torch.zeros(2, dtype=torch.int32)
    got = trunk.attention_rows(torch.zeros(0, 128, dtype=torch.bfloat16), affine(8 * 64, 128), affine(128, 4 * 64),
                               attention.KVCache.empty(1, 2, 64, device="cpu"), cu[:1, None], cu[:1], cu=cu,
                               prompt=(cu, 0) if prompt == "later" else prompt)
    assert got.shape == (0, 128)


def test_a_cache_of_no_heads_is_refused():
    cache, i = attention.KVCache.empty(1, 0, 64, device="cpu"), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="0 key heads"):
        attention.attend_rows(torch.zeros(1, 2, 64, dtype=torch.float16), cache, i[None], i)
    with pytest.raises(ValueError, match="0 key heads"):
        attention.prompt_rows(torch.zeros(1, 2, 64, dtype=torch.float16), *[torch.zeros(1, 0, 64, dtype=torch.float16)] * 2, i)


@pytest.mark.parametrize("most", [-1, 0, 1, 3, 2 ** 31 - 1, 2 ** 31, 2 ** 32 + 1, 10 ** 30])
@pytest.mark.parametrize("longest", [-1, 5, 2 ** 31, 2 ** 32, 10 ** 30])
def test_any_most_rows_and_longest_size_a_launch(monkeypatch, built_lib, most, longest):
    """What they are worth to a launch is bounded by the rows and the table, so that no value passes an int."""
    sizes = []
    monkeypatch.setattr(attention, "_device", lambda *a: 0)
    monkeypatch.setattr(attention, "_launch", lambda dev, name, *args: sizes.append(args))
    cache = attention.KVCache.empty(1, 1, 64, device="cpu")
    attention.attend_rows(torch.zeros(3, 2, 64, dtype=torch.float16), cache, torch.zeros(1, 20, dtype=torch.int32), CU[1:],
                          cu=CU, most_rows=most, longest=longest)
    rows, tokens = sizes[0][19:21]
    assert rows == min(max(most, 1), 3) and tokens == min(max(longest, 1), 20 * 64)
    assert sizes[0][23] == built_lib.lmoe_kv_attend_workspace_bytes(3, 2, 1, 64, 1, rows, tokens)


P = ctypes.c_void_p(16)  # never dereferenced: every call below is refused while its arguments are checked
ODD = ctypes.c_void_p(24)


def refused(L, code, word, name, *args):
    rc = getattr(L, name)(*args, None)
    assert rc == code and word in L.lmoe_error(), (rc, L.lmoe_error())


def test_entry_points_refuse(built_lib):
    L = built_lib

    def rope(x=P, dt=1, st=64, pos=P, freq=P, n=32, T=2, h=1, D=64, out=P):
        return x, dt, st, 64, pos, 0, freq, n, T, h, D, 0, 1.0, out, 64, 64

    refused(L, _lib.EINVAL, b"dtype", "lmoe_rope_rows", *rope(dt=3))
    refused(L, _lib.ESHAPE, b"pairs", "lmoe_rope_rows", *rope(n=33))
    refused(L, _lib.ESHAPE, b"heads of", "lmoe_rope_rows", *rope(D=1026))
    refused(L, _lib.ESHAPE, b"rows", "lmoe_rope_rows", *rope(T=-1))
    refused(L, _lib.EINVAL, b"null", "lmoe_rope_rows", *rope(pos=None))
    refused(L, _lib.EINVAL, b"null", "lmoe_rope_rows", *rope(freq=None))
    assert L.lmoe_rope_rows(*rope(T=0, x=None), None) == 0

    def append(q=P, k=P, v=P, dt=1, T=2, heads=1, D=64, cu=P, B=1, width=1, pages=1, page=64, n=32, inter=0, st=128, codes=P,
               q_out=P):
        return (q, st, 64, 1, k, st, 64, v, st, 64, dt, T, heads, D, cu, P, B, P, width, codes, P, P, P, pages, page, P, n, inter,
                1.0, q_out, None)

    refused(L, _lib.EINVAL, b"dtype", "lmoe_kv_append", *append(dt=7))
    refused(L, _lib.ESHAPE, b"channels", "lmoe_kv_append", *append(D=96, n=0))
    refused(L, _lib.ESHAPE, b"tokens", "lmoe_kv_append", *append(page=16))
    refused(L, _lib.ESHAPE, b"pairs", "lmoe_kv_append", *append(n=12))
    refused(L, _lib.ESHAPE, b"pairs", "lmoe_kv_append", *append(n=6, inter=1))
    refused(L, _lib.ESHAPE, b"pairs", "lmoe_kv_append", *append(n=40))
    refused(L, _lib.ESHAPE, b"offsets", "lmoe_kv_append", *append(cu=None))
    refused(L, _lib.ESHAPE, b"pages", "lmoe_kv_append", *append(pages=0))
    refused(L, _lib.EINVAL, b"null", "lmoe_kv_append", *append(k=None))
    refused(L, _lib.EINVAL, b"null", "lmoe_kv_append", *append(q_out=None))
    refused(L, _lib.EALIGN, b"aligned", "lmoe_kv_append", *append(k=ODD))
    refused(L, _lib.EALIGN, b"aligned", "lmoe_kv_append", *append(st=68))
    refused(L, _lib.EALIGN, b"aligned", "lmoe_kv_append", *append(codes=ODD))
    assert L.lmoe_kv_append(*append(T=0), None) == 0

    def read(pages=1, page=64, heads=1, D=64, B=1, total=2, k=P, dt=1):
        return P, P, P, P, pages, page, heads, D, P, 1, P, B, total, k, P, dt

    refused(L, _lib.EINVAL, b"dtype", "lmoe_kv_read", *read(dt=9))
    refused(L, _lib.ESHAPE, b"rows", "lmoe_kv_read", *read(total=-1))
    refused(L, _lib.ESHAPE, b"channels", "lmoe_kv_read", *read(D=32))
    refused(L, _lib.EINVAL, b"null", "lmoe_kv_read", *read(k=None))
    refused(L, _lib.EALIGN, b"aligned", "lmoe_kv_read", *read(k=ODD))

    def attend(q=P, dt=1, st=64, T=2, qh=2, h=1, D=64, cu=P, B=1, pages=1, page=64, most=1, longest=8192, ws=P, wsb=1 << 30):
        return (q, dt, st, 64, T, qh, h, D, cu, P, B, P, 1, P, P, P, P, pages, page, most, longest, 0.125, ws, wsb, P)

    refused(L, _lib.EINVAL, b"dtype", "lmoe_kv_attend", *attend(dt=0))
    refused(L, _lib.ESHAPE, b"query heads", "lmoe_kv_attend", *attend(qh=3, h=2))
    refused(L, _lib.ESHAPE, b"channels", "lmoe_kv_attend", *attend(D=192))
    refused(L, _lib.ESHAPE, b"tokens", "lmoe_kv_attend", *attend(page=256))
    refused(L, _lib.ESHAPE, b"sequences", "lmoe_kv_attend", *attend(longest=0))
    refused(L, _lib.ESHAPE, b"offsets", "lmoe_kv_attend", *attend(cu=None))
    refused(L, _lib.EINVAL, b"null", "lmoe_kv_attend", *attend(q=None))
    refused(L, _lib.EALIGN, b"aligned", "lmoe_kv_attend", *attend(st=65))
    refused(L, _lib.EWORKSPACE, b"workspace", "lmoe_kv_attend", *attend(wsb=16))
    refused(L, _lib.EWORKSPACE, b"workspace", "lmoe_kv_attend", *attend(ws=None))

    def prompt(q=P, k=P, st=64, kst=64, dt=1, T=2, U=2, qh=1, h=1, D=64, cu=P, B=1, ws=P, wsb=1 << 30):
        return q, st, 64, k, kst, 64, P, 64, 64, dt, T, U, qh, h, D, cu, P, B, 0.125, ws, wsb, P

    refused(L, _lib.EINVAL, b"dtype", "lmoe_prompt_attend", *prompt(dt=0))
    refused(L, _lib.ESHAPE, b"channels", "lmoe_prompt_attend", *prompt(D=80))
    refused(L, _lib.ESHAPE, b"query heads", "lmoe_prompt_attend", *prompt(qh=3, h=2))
    refused(L, _lib.ESHAPE, b"sequence", "lmoe_prompt_attend", *prompt(B=0))
    refused(L, _lib.EINVAL, b"null", "lmoe_prompt_attend", *prompt(cu=None))
    refused(L, _lib.EALIGN, b"aligned", "lmoe_prompt_attend", *prompt(q=ODD))
    refused(L, _lib.ESHAPE, b"apart", "lmoe_prompt_attend", *prompt(kst=1 << 23))
    refused(L, _lib.EWORKSPACE, b"workspace", "lmoe_prompt_attend", *prompt(U=8192, wsb=16))
    refused(L, _lib.EWORKSPACE, b"workspace", "lmoe_prompt_attend", *prompt(U=8192, ws=None))
    assert L.lmoe_prompt_attend(*prompt(T=0), None) == 0


def test_attend_workspace(built_lib):
    need = built_lib.lmoe_kv_attend_workspace_bytes
    assert need(1, 16, 16, 128, 1, 1, 100) == 0                       # each sequence whole: nothing to join
    assert need(1, 32, 4, 128, 1, 1, 8192) == 256 * 2 * 16 * 130 * 4 + 32 * 8   # 64 units of 4 heads: two places each
    assert need(64, 32, 4, 128, 64, 1, 8192) == 512 * 2 * 16 * 130 * 4 + 64 * 32 * 8  # at most two workgroups a CU
    assert need(1, 3, 2, 128, 1, 1, 8192) == 0                        # refused shapes ask for nothing
    need = built_lib.lmoe_prompt_attend_workspace_bytes
    assert need(8192, 8192, 32, 4, 128, 1) == 0 and need(300, 300, 4, 4, 128, 1) == 0
    assert need(100, 8100, 28, 4, 128, 1) == 16 * 100 * 28 * 132 * 4 + 100 * 28 * 4  # 28 workgroups: 18 chunks, 512 keys at least


def test_workspace_of_the_largest_sizes(built_lib):
    """longest and most_rows of an int's end size a launch like any other: at most two workgroups a CU, two places each."""
    need = built_lib.lmoe_kv_attend_workspace_bytes
    for longest in (1 << 30, 2 ** 31 - 127, 2 ** 31 - 1):
        for most in (1, 2 ** 31 - 1):
            assert need(1, 32, 4, 128, 1, most, longest) == 512 * 2 * 16 * 130 * 4 + 32 * 8


@pytest.mark.parametrize("page", [32, 64, 128])
def test_tables_of_places_past_an_int_are_refused(built_lib, page):
    """A table whose last page ends past 2^31 - 1: that page's tokens would not be written."""
    wide = (1 << 31) // page
    for name, *args in (("lmoe_kv_append", None, 64, 64, 0, P, 64, 64, P, 64, 64, 1, 1, 1, 64, P, P, 1, P, wide, P, P, P, P, 1, page, P,
                         0, 0, 1.0, None, None),
                        ("lmoe_kv_read", P, P, P, P, 1, page, 1, 64, P, wide, P, 1, 1, P, P, 1),
                        ("lmoe_kv_attend", P, 1, 64, 64, 1, 1, 1, 64, P, P, 1, P, wide, P, P, P, P, 1, page, 1, 100, 0.1, P, 0, P)):
        refused(built_lib, _lib.ESHAPE, b"a table of", name, *args)


def test_more_than_a_launch_takes_is_refused(built_lib):
    """Grids of 2^24 workgroups of 256 and more, which the runtime would cut to what is left of them in 32 bits."""
    def check(name, *args):
        refused(built_lib, _lib.ESHAPE, b"than a launch takes", name, *args)

    for t in (8 * (2 ** 24 - 1) + 1, 2 ** 31 - 1):
        check("lmoe_rope_rows", P, 1, 64, 64, P, 0, P, 32, t, 1, 64, 0, 1.0, P, 64, 64)
    for t, b, cu in ((100, 2 ** 22, P), (2 ** 23, 2 ** 23, None), (2 ** 31 - 1, 1, P)):
        check("lmoe_kv_append", None, 64, 64, 0, P, 64, 64, P, 64, 64, 1, t, 1, 64, cu, P, b, P, 1, P, P, P, P, 1, 64, P, 0, 0, 1.0,
              None, None)
    for total in (16 * (2 ** 24 - 1) + 1, 2 ** 31 - 1):
        check("lmoe_kv_read", P, P, P, P, 1, 64, 1, 64, P, 1, P, 1, total, P, P, 1)
    check("lmoe_prompt_attend", P, 64, 64, P, 64, 64, P, 64, 64, 1, 2, 2, 32, 4, 64, P, P, 2 ** 19, 0.1, P, 0, P)


@pytest.mark.parametrize("heads", [(1 << 20) + 1, 1 << 24, 2 ** 31 - 1])
def test_rows_of_more_channels_than_an_int_counts_are_refused(built_lib, heads):
    refused(built_lib, _lib.ESHAPE, b"heads of 1024", "lmoe_rope_rows", P, 1, 64, 1024, P, 0, P, 32, 2, heads, 1024, 0, 1.0, P, 64, 1024)
    refused(built_lib, _lib.ESHAPE, b"query heads of 256", "lmoe_kv_append", P, 256, 256, max(heads, 1 << 22), P, 64, 64, P, 64, 64, 1, 2,
            1, 256, P, P, 1, P, 1, P, P, P, P, 1, 64, P, 0, 0, 1.0, P, None)


@pytest.mark.parametrize("unit,spare", [(32, 2), (64, 2), (128, 2), (128, 1)])
def test_every_page_and_tile_has_a_workgroup(unit, spare):
    """Sequence b's workgroups begin at cu[b] // unit + spare b. With spare 2 that is room for every page that its rows can
    touch, wherever they begin in the first (k_append); with spare 1 for every tile of unit rows (k_prompt)."""
    rng = np.random.default_rng(unit + spare)
    for _ in range(200):
        n = rng.choice([0, 1, 2, unit - 1, unit, unit + 1, 3 * unit + 5], 8)
        cu = np.concatenate([[0], np.cumsum(n)])
        first = cu // unit + spare * np.arange(9)
        for b in range(8):
            start = rng.integers(0, unit) if spare == 2 else 0
            touched = 0 if n[b] == 0 else (start + n[b] - 1) // unit - start // unit + 1
            assert touched <= first[b + 1] - first[b]
        assert first[8] == cu[8] // unit + spare * 8                  # what the host launches
