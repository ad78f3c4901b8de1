"""The attention of the trunk's rows, as cases that can be timed and compared: rotary positions, appending keys and
values to a paged 8-bit cache, attention of single tokens (or a few draft rows) over that cache, and attention over whole
packed prompts.

Kinds (key "kind") and the calls of larder_amd.attention they make:
  rope     rope_rows: rotary positions of T rows
  append   append_rows, and read_rows of the pages it touched, so that the cache comes back as the values it stands for
  attend   attend_rows: the newest rows of each sequence over the cache
  prompt   prompt_rows: packed sequences, causal, each row over its sequence's keys

The cache: codes float8_e4m3fn [pages, heads, page, width] of keys and of values, and a power-of-two float32 scale for each
page and head. A page's scale is the least power of two (2^-100 or more) that brings its largest finite magnitude to 448 or
less; a page that held tokens before keeps the larger of its old and the new scale, and its codes are restated in that.
Lengths of a case's sequences follow from its "seqs", "longest" and "mix" alone.
"""
import math
import random

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
# (query heads, key heads, width, rotated width): one key head a query head, groups of 8 and of an odd 7, few wide heads
# rotated in part, small heads
HEADS = {"16x16x128": (16, 16, 128, 128), "32x4x128": (32, 4, 128, 128), "28x4x128": (28, 4, 128, 128),
         "16x2x256": (16, 2, 256, 64), "32x2x256": (32, 2, 256, 64), "12x4x64": (12, 4, 64, 64), "8x8x64": (8, 8, 64, 32)}


def listed():
    return [
        # one token's queries: nothing but latency
        dict(name="rope_1_token", kind="rope", T=1, heads="32x4x128", dtype="bf16", interleaved=False, at=5000, factor=1.0),
        # a whole prompt chunk far into a stretched context, neighbouring pairs
        dict(name="rope_8192_far", kind="rope", T=8192, heads="32x4x128", dtype="f16", interleaved=True, at=100000,
             factor=4.0),
        # a decode step of 64 running sequences
        dict(name="append_batch_64", kind="append", heads="32x4x128", dtype="bf16", page=64, seqs=64, new=1, longest=4096,
             mix=1, interleaved=False, factor=1.0),
        # a packed prefill of several prompts, the first continued from an earlier chunk, heads rotated in part
        dict(name="append_prompts", kind="append", heads="16x2x256", dtype="f16", page=64, seqs=9, new=2048, longest=4096,
             mix=2, interleaved=False, factor=1.0),
        # one token of a short chat: the smallest work, launches and latency
        dict(name="attend_short", kind="attend", heads="16x16x128", dtype="f16", page=64, seqs=1, rows=1, longest=201, mix=3),
        # one token of a long context
        dict(name="attend_1_long", kind="attend", heads="32x4x128", dtype="bf16", page=64, seqs=1, rows=1, longest=131072,
             mix=4),
        # a speculative decoder's verify rows of a few sequences, wide heads, small pages
        dict(name="attend_drafts", kind="attend", heads="16x2x256", dtype="f16", page=32, seqs=4, rows=5, longest=3001,
             mix=5),
        # continuous batching: 64 sequences of different lengths
        dict(name="attend_batch_64", kind="attend", heads="32x4x128", dtype="bf16", page=64, seqs=64, rows=1, longest=16384,
             mix=6),
        # a few short, odd prompts packed
        dict(name="prompt_short", kind="prompt", heads="16x16x128", dtype="bf16", seqs=3, longest=333, past=0, mix=7),
        # a chunk of a long prompt, over the keys before it too
        dict(name="prompt_chunk", kind="prompt", heads="28x4x128", dtype="bf16", seqs=1, longest=1024, past=7000, mix=8),
        # many prompts packed, wide heads
        dict(name="prompt_packed", kind="prompt", heads="16x2x256", dtype="f16", seqs=12, longest=2500, past=0, mix=9),
        # one full prompt
        dict(name="prompt_8192", kind="prompt", heads="32x4x128", dtype="bf16", seqs=1, longest=8192, past=0, mix=10),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "append", "append", "attend", "attend", "attend", "prompt", "prompt", "prompt"])
    heads = rng.choice(sorted(HEADS))
    mix = rng.randrange(1 << 20)
    dtype = rng.choice(["f16", "bf16"])
    interleaved, factor = rng.random() < 0.5, rng.choice([1.0, 1.0, 2.0, 8.0])
    if kind == "rope":
        return dict(kind=kind, T=_log_int(rng, 1, 8192), heads=heads, dtype=rng.choice(["f16", "bf16", "f32"]),
                    interleaved=interleaved, at=_log_int(rng, 1, 1000000), factor=factor)
    page = rng.choice([32, 64, 128])
    if kind == "append":
        new = rng.choice([1, 1, 4, _log_int(rng, 5, 2048)])
        return dict(kind=kind, heads=heads, dtype=dtype, page=page, seqs=_log_int(rng, 1, 64 if new < 5 else 9), new=new,
                    longest=_log_int(rng, max(64, new), 4096), mix=mix, interleaved=interleaved, factor=factor)
    if kind == "attend":
        seqs, rows = _log_int(rng, 1, 64), rng.choice([1, 1, 1, 2, 5, 16])
        return dict(kind=kind, heads=heads, dtype=dtype, page=page, seqs=seqs, rows=rows, mix=mix,
                    longest=_log_int(rng, 40, min(131072, 262144 // seqs)))
    seqs, past = rng.choice([(1, 0), (1, _log_int(rng, 1, 8000)), (_log_int(rng, 2, 16), 0)])
    case = dict(kind=kind, heads=heads, dtype=dtype, seqs=seqs, past=past, longest=_log_int(rng, 17, 8192), mix=mix)
    while work(case)["flops"] > 5e11:
        case["longest"] = case["longest"] * 2 // 3
    return case


# ---- sizes -----------------------------------------------------------------------------------------------------

def _lengths(case):
    """The sequences' lengths: one of the longest, the others spread below it, over the logarithm."""
    rng = random.Random(case["mix"])
    n = case["longest"]
    return [n] + [_log_int(rng, max(1, n // 16), n) for _ in range(case["seqs"] - 1)]


def _append_sizes(case):
    """(tokens held before, tokens appended) of each sequence: one token each in a decode step; in a prefill the first is a
    later chunk of its prompt and the others begin."""
    if case["new"] < 5:
        return [n - 1 for n in _lengths(case)], [case["new"]] * case["seqs"]
    new = _lengths(dict(case, longest=case["new"]))
    return [case["longest"] - case["new"]] + [0] * (case["seqs"] - 1), new


def _visible(nq, nk):
    """The (row, key) pairs of a causal sequence aligned at its end, nk >= nq."""
    return nq * (nk - nq) + nq * (nq + 1) // 2


def work(case):
    hq, hk, d, rot = HEADS[case["heads"]]
    size = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "rope":
        t = case["T"]
        return {"bytes": 2 * t * hq * d * size + 4 * t + 4 * rot, "flops": 3 * t * hq * rot}
    if case["kind"] == "append":
        old, new = _append_sizes(case)
        t, p = sum(new), case["page"]
        # the pages' tokens come back in 16 bits; those that were there before are read in 8
        touched = sum(o + n - o // p * p for o, n in zip(old, new))
        rows = t * (2 * hq + 3 * hk) * d * size + 2 * t * hk * d
        return {"bytes": rows + 2 * (3 * touched - t) * hk * d, "flops": 3 * t * (hq + hk) * rot + 2 * t * hk * d}
    if case["kind"] == "attend":
        n, r = sum(max(x, case["rows"]) for x in _lengths(case)), case["seqs"] * case["rows"]
        return {"bytes": 2 * n * hk * d + 2 * r * hq * d * size, "flops": 4 * n * case["rows"] * hq * d}
    qs = _lengths(case)
    ks = [n + case["past"] for n in qs]
    return {"bytes": (2 * sum(qs) * hq + 2 * sum(ks) * hk) * d * size,
            "flops": 4 * hq * d * sum(_visible(a, b) for a, b in zip(qs, ks))}


# ---- inputs ----------------------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _cu(lengths):
    return _ints([sum(lengths[:i]) for i in range(len(lengths) + 1)])


def _frequencies(case, rot):
    """Radians a position of each pair, in 64 bits, positions interpolated by the case's factor."""
    i = torch.arange(0, rot, 2, dtype=torch.float64, device="cuda")
    return (1.0 / 1e6 ** (i / rot)) / case["factor"]


def _channels(gen, hk, d):
    """Keys have channels that stand out; their spread."""
    return torch.exp(0.5 * _normal(gen, hk, d))


def _table(gen, counts):
    """A table of page numbers [sequences, most pages] in no order, no page twice, and how many pages there are."""
    n = sum(counts) + 3
    order = torch.randperm(n, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros((len(counts), max(counts)), dtype=torch.int32, device="cuda")
    at = 0
    for b, c in enumerate(counts):
        table[b, :c] = order[at:at + c]
        at += c
    return table, n


def _pages(gen, n, hk, page, d, spread):
    """n pages of random tokens in the cache's form, and their scales, some hundred pages at a time."""
    codes = torch.empty((n, hk, page, d), dtype=torch.float8_e4m3fn, device="cuda")
    scales = torch.empty((n, hk), dtype=torch.float32, device="cuda")
    for at in range(0, n, 512):
        x = _normal(gen, min(512, n - at), hk, page, d)
        x = x if spread is None else x * spread[:, None, :]
        s = _need(x.abs().amax((2, 3)))
        codes[at:at + 512] = (x / s[..., None, None]).to(torch.float8_e4m3fn)
        scales[at:at + 512] = s
    return codes, scales


def prepare(case, seed):
    hq, hk, d, rot = HEADS[case["heads"]]
    gen, dt = _gen(seed), DTYPES[case["dtype"]]
    s = dict(case)
    if case["kind"] == "rope":
        t = case["T"]
        s["x"] = _normal(gen, t, hq, d).to(dt)
        s["positions"] = torch.arange(case["at"], case["at"] + t, dtype=torch.int32, device="cuda")
        s["freq"] = _frequencies(case, rot)
        return s
    if case["kind"] == "prompt":
        qs = _lengths(case)
        ks = [n + case["past"] for n in qs]
        spread = _channels(gen, hk, d)
        s["q"] = _normal(gen, sum(qs), hq, d).to(dt)
        s["k"] = (_normal(gen, sum(ks), hk, d) * spread).to(dt)
        s["v"] = _normal(gen, sum(ks), hk, d).to(dt)
        s["cu"], s["cu_k"] = _cu(qs), _cu(ks)
        return s
    page, spread = case["page"], _channels(gen, hk, d)
    if case["kind"] == "attend":
        lens = [max(n, case["rows"]) for n in _lengths(case)]
        s["table"], n = _table(gen, [-(-x // page) for x in lens])
        s["lens"], s["rows_cu"] = _ints(lens), _cu([case["rows"]] * case["seqs"])
        s["most"] = max(lens)
        s["q"] = _normal(gen, case["seqs"] * case["rows"], hq, d).to(dt)
    else:
        old, new = _append_sizes(case)
        lens = [a + b for a, b in zip(old, new)]
        s["table"], n = _table(gen, [-(-x // page) for x in lens])
        s["lens"], s["rows_cu"], s["freq"] = _ints(lens), _cu(new), _frequencies(case, rot)
        # the trunk's product gives q, k and v of a token side by side
        x = _normal(gen, sum(new), hq + 2 * hk, d)
        x[:, hq:hq + hk] *= spread
        s["q"], s["k"], s["v"] = x.to(dt).split([hq, hk, hk], 1)
        # the pages the rows fall into, which come back
        first = [a // page for a in old]
        s["back_table"] = torch.zeros((len(lens), max(-(-x // page) - f for x, f in zip(lens, first))), dtype=torch.int32,
                                      device="cuda")
        for b, (x, f) in enumerate(zip(lens, first)):
            c = -(-x // page) - f
            s["back_table"][b, :c] = s["table"][b, f:f + c]
        back = [x - f * page for x, f in zip(lens, first)]
        s["back_cu"], s["back_total"] = _cu(back), sum(back)
    s["k_pages"], s["k_scale"] = _pages(gen, n, hk, page, d, spread)
    s["v_pages"], s["v_scale"] = _pages(gen, n, hk, page, d, None)
    return s


# ---- the plain forms -------------------------------------------------------------------------------------------

def _need(most):
    """The least power of two, 2^-100 or more, that brings `most` to 448 or less."""
    m, e = torch.frexp(most)
    e = torch.where(most > 0, e - 9 + (m > 0.875).to(e.dtype), -100).clamp(min=-100)
    return ((e + 127) << 23).view(torch.float32)  # 2^e by its bits


def _rotated(x, positions, freq, interleaved):
    """x [T, heads, width] float32, its first 2 len(freq) channels rotated; angles in 64 bits."""
    angle = positions.to(torch.float64)[:, None, None] * freq
    c, s = torch.cos(angle).to(torch.float32), torch.sin(angle).to(torch.float32)
    r = 2 * freq.numel()
    if interleaved:
        u, w = x[..., 0:r:2], x[..., 1:r:2]
        y = torch.stack([u * c - w * s, w * c + u * s], -1).flatten(-2)
    else:
        u, w = x[..., :r // 2], x[..., r // 2:r]
        y = torch.cat([u * c - w * s, w * c + u * s], -1)
    return torch.cat([y, x[..., r:]], -1)


def _owner(cu, total):
    """The sequence of each packed row, and the row's place in it."""
    i = torch.arange(total, dtype=torch.int32, device="cuda")
    b = torch.searchsorted(cu, i, right=True).long() - 1
    return b, i.long() - cu.long()[b]


def _into_pages(codes, scales, x, page_of, at, fresh, touched):
    """Writes the rows x [T, heads, width] float32 at (page, place) into codes and scales, in place."""
    most = torch.zeros_like(scales).index_reduce_(0, page_of, x.abs().amax(-1), "amax")
    old = torch.where(fresh[:, None], torch.zeros_like(scales), scales)
    new = torch.maximum(old, _need(most))[touched]
    raw = codes.view(torch.uint8)
    held = raw[touched].view(torch.float8_e4m3fn).to(torch.float32) * (old[touched] / new)[..., None, None]
    raw[touched] = held.to(torch.float8_e4m3fn).view(torch.uint8)
    scales[touched] = new
    raw[page_of, :, at] = (x / scales[page_of][..., None]).to(torch.float8_e4m3fn).view(torch.uint8)


def _from_pages(codes, scales, table, cu, total):
    """Packed rows [total, heads, width] float32 of the sequences' first cu[b + 1] - cu[b] tokens."""
    b, i = _owner(cu, total)
    page = codes.shape[2]
    p = table.long()[b, i // page]
    return codes.view(torch.uint8)[p, :, i % page].view(torch.float8_e4m3fn).to(torch.float32) * scales[p][..., None]


def _plain_append(s):
    page, total = s["k_pages"].shape[2], s["q"].shape[0]
    b, i = _owner(s["rows_cu"], total)
    n = (s["rows_cu"][1:] - s["rows_cu"][:-1]).long()
    pos = s["lens"].long()[b] - n[b] + i
    q = _rotated(s["q"].to(torch.float32), pos, s["freq"], s["interleaved"])
    k = _rotated(s["k"].to(torch.float32), pos, s["freq"], s["interleaved"])
    page_of = s["table"].long()[b, pos // page]
    pages = s["k_scale"].shape[0]
    fresh = torch.zeros(pages, dtype=torch.bool, device="cuda")
    fresh[page_of[pos % page == 0]] = True
    touched = torch.unique(page_of)
    _into_pages(s["k_pages"], s["k_scale"], k, page_of, pos % page, fresh, touched)
    _into_pages(s["v_pages"], s["v_scale"], s["v"].to(torch.float32), page_of, pos % page, fresh, touched)
    dt = s["q"].dtype
    back = [_from_pages(c, e, s["back_table"], s["back_cu"], s["back_total"]).to(dt)
            for c, e in ((s["k_pages"], s["k_scale"]), (s["v_pages"], s["v_scale"]))]
    return q.to(dt), k.to(dt), back[0], back[1], s["k_scale"], s["v_scale"]


def _softmax_rows(scores, seen):
    """softmax over the last axis where `seen`; rows that see nothing are zero."""
    scores = scores.masked_fill(~seen, float("-inf"))
    m = scores.amax(-1, keepdim=True).clamp(min=torch.finfo(scores.dtype).min)
    e = torch.exp(scores - m)
    return e / e.sum(-1, keepdim=True).clamp(min=torch.finfo(scores.dtype).tiny)


def _gathered(codes, scales, table):
    """float32 [sequences, heads, most tokens, width] of every page in the table."""
    x = codes.view(torch.uint8)[table.long()].view(torch.float8_e4m3fn).to(torch.float32)
    x = x * scales[table.long()][..., None, None]
    return x.transpose(1, 2).flatten(2, 3)


def _plain_attend(s):
    hq, hk, d, _ = HEADS[s["heads"]]
    b, r, g = s["seqs"], s["rows"], hq // hk
    k, v = _gathered(s["k_pages"], s["k_scale"], s["table"]), _gathered(s["v_pages"], s["v_scale"], s["table"])
    q = s["q"].to(torch.float32).view(b, r, hk, g, d).permute(0, 2, 1, 3, 4).reshape(b, hk, r * g, d)
    scores = (q @ k.transpose(2, 3)).view(b, hk, r, g, -1) / math.sqrt(d)
    last = s["lens"].long()[:, None] - r + torch.arange(r, device="cuda")
    seen = torch.arange(k.shape[2], device="cuda") <= last[..., None]
    p = _softmax_rows(scores, seen[:, None, :, None, :])
    o = (p.view(b, hk, r * g, -1) @ v).view(b, hk, r, g, d)
    return o.permute(0, 2, 1, 3, 4).reshape(b * r, hq, d).to(s["q"].dtype)


def _plain_prompt(s):
    hq, hk, d, _ = HEADS[s["heads"]]
    t, u, g = s["q"].shape[0], s["k"].shape[0], hq // hk
    b, i = _owner(s["cu"], t)
    c, j = _owner(s["cu_k"], u)
    nq, nk = (s["cu"][1:] - s["cu"][:-1]).long(), (s["cu_k"][1:] - s["cu_k"][:-1]).long()
    seen = (b[:, None] == c) & (j <= (i + (nk - nq)[b])[:, None])
    q = s["q"].to(torch.float32).view(t, hk, g, d).permute(1, 2, 0, 3).reshape(hk, g * t, d)
    k, v = s["k"].to(torch.float32).transpose(0, 1), s["v"].to(torch.float32).transpose(0, 1)
    scores = (q @ k.transpose(1, 2)).view(hk, g, t, u) / math.sqrt(d)
    p = _softmax_rows(scores, seen)
    o = (p.view(hk, g * t, u) @ v).view(hk, g, t, d)
    return o.permute(2, 0, 1, 3).reshape(t, hq, d).to(s["q"].dtype)


# ---- one pass --------------------------------------------------------------------------------------------------

def _own(s):
    from larder_amd import attention
    if s["kind"] == "rope":
        return attention.rope_rows(s["x"], s["positions"], s["freq"], interleaved=s["interleaved"])
    if s["kind"] == "prompt":
        return attention.prompt_rows(s["q"], s["k"], s["v"], s["cu"], cu_k=s["cu_k"])
    cache = attention.KVCache(s["k_pages"], s["k_scale"], s["v_pages"], s["v_scale"])
    if s["kind"] == "attend":
        return attention.attend_rows(s["q"], cache, s["table"], s["lens"], cu=s["rows_cu"], most_rows=s["rows"],
                                     longest=s["most"])
    q, k = attention.append_rows(cache, s["q"], s["k"], s["v"], s["table"], s["lens"], cu=s["rows_cu"], freq=s["freq"],
                                 interleaved=s["interleaved"], keys=True)
    back = attention.read_rows(cache, s["back_table"], s["back_cu"], s["back_total"], dtype=s["q"].dtype)
    return q, k, back[0], back[1], s["k_scale"], s["v_scale"]


def run(state):
    if own:
        return _own(state)
    if state["kind"] == "rope":
        x = state["x"]
        return _rotated(x.to(torch.float32), state["positions"], state["freq"], state["interleaved"]).to(x.dtype)
    return {"append": _plain_append, "attend": _plain_attend, "prompt": _plain_prompt}[state["kind"]](state)


# ---- the answers in 64 bits ------------------------------------------------------------------------------------

def _exact_rope(x, positions, freq, interleaved):
    x = x.to(torch.float64)
    r = 2 * freq.numel()
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), positions.to(torch.float64)[:, None] * freq)
    pair = x[..., :r].unflatten(-1, (-1, 2) if interleaved else (2, -1))
    axis = -1 if interleaved else -2
    z = torch.complex(*pair.unbind(axis)) * turn[:, None, :]
    x[..., :r] = torch.stack([z.real, z.imag], axis).flatten(-2)
    return x


def _exact_codes(x):
    """x rounded to the nearest e4m3 value (ties to even), as float64; |x| <= 448."""
    e = torch.clamp(torch.frexp(x)[1] - 1, min=-6) - 3
    step = ((e.to(torch.int64) + 1023) << 52).view(torch.float64)
    return torch.round(x / step) * step


def _exact_append(s):
    page = s["k_pages"].shape[2]
    cu, lens = s["rows_cu"].tolist(), s["lens"].tolist()
    pos = torch.cat([torch.arange(n - (b - a), n, device="cuda") for n, a, b in zip(lens, cu, cu[1:])])
    q, k = (_exact_rope(s[m], pos, s["freq"], s["interleaved"]) for m in ("q", "k"))
    back, scales = [], []
    for rows, codes, held in ((k, s["k_pages"], s["k_scale"]), (s["v"].to(torch.float64), s["v_pages"], s["v_scale"])):
        scale, out = held.to(torch.float64), []
        for b, n in enumerate(lens):
            start = n - (cu[b + 1] - cu[b])
            for p in range(start // page, -(-n // page)):
                number = int(s["table"][b, p])
                lo, hi = max(start, p * page), min(n, (p + 1) * page)
                new = rows[cu[b] + lo - start:cu[b] + hi - start]
                before = codes[number, :, :lo - p * page].to(torch.float64).transpose(0, 1) * scale[number][:, None]
                top = new.abs().amax((0, 2))
                m, e = torch.frexp((top / 448).clamp(min=2.0 ** -100))
                need = (((e - (m == 0.5).to(e.dtype)).to(torch.int64) + 1023) << 52).view(torch.float64)
                scale[number] = need if lo == p * page else torch.maximum(need, scale[number])
                both = torch.cat([before, new])
                out.append(_exact_codes(both / scale[number][:, None]) * scale[number][:, None])
        back.append(torch.cat(out))
        scales.append(scale)
    return q, k, back[0], back[1], scales[0], scales[1]


def _exact_attention(q, k, v, past):
    """q [n, hq, d] over k, v [m, hk, d] float64: row i sees keys 0 .. i + past."""
    n, hq, d = q.shape
    g = hq // k.shape[1]
    seen = torch.arange(k.shape[0], device="cuda") <= torch.arange(n, device="cuda")[:, None] + past
    out = torch.empty_like(q)
    for h in range(hq):
        x = (q[:, h] @ k[:, h // g].t()) / math.sqrt(d)
        out[:, h] = torch.softmax(x.masked_fill(~seen, float("-inf")), -1) @ v[:, h // g]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rope":
        return _exact_rope(s["x"], s["positions"], s["freq"], s["interleaved"])
    if case["kind"] == "append":
        return _exact_append(s)
    q, out = s["q"].to(torch.float64), []
    if case["kind"] == "prompt":
        cu, cu_k = s["cu"].tolist(), s["cu_k"].tolist()
        k, v = s["k"].to(torch.float64), s["v"].to(torch.float64)
        for a, b, c, e in zip(cu, cu[1:], cu_k, cu_k[1:]):
            out.append(_exact_attention(q[a:b], k[c:e], v[c:e], (e - c) - (b - a)))
        return torch.cat(out)
    r, page = case["rows"], case["page"]
    for b, n in enumerate(s["lens"].tolist()):
        pages = s["table"][b, :-(-n // page)].long()
        k, v = ((c.view(torch.uint8)[pages].view(torch.float8_e4m3fn).to(torch.float64) * e[pages][..., None, None])
                .transpose(1, 2).flatten(0, 1)[:n] for c, e in ((s["k_pages"], s["k_scale"]), (s["v_pages"], s["v_scale"])))
        out.append(_exact_attention(q[b * r:(b + 1) * r], k, v, n - r))
    return torch.cat(out)
