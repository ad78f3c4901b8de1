"""What a serving step does around the trunk's products, as cases that can be timed and compared: root-mean-square norms with
the residual's addition (in 16 bits, or 8 with scales), the pages of the 8-bit cache given, shared, copied, freed and
compacted, and attention of chunks of new rows over that cache's pages.

Kinds (key "kind") and the calls they make:
  norm     trunk.norm_rows: rows of the residual stream, or heads of a product before their rotation; in 8 bits the codes are
           read back by trunk.read_codes, so that the rows come as the values they stand for
  step     pages.free_pages and pages.take_pages: finished sequences leave, the others' newest rows get their pages, shared pages
           that would be written are copied (pages.copy_pages); the copies are read back
  beam     pages.fork_pages, then as a step: the sequences go on from others' histories
  compact  pages.compact_pages and pages.copy_pages: held pages moved into the lowest numbers; the moved pages are read back
  chunk    attention.chunk_rows: a chunk of new rows of each sequence over its cached tokens, causal

A norm's row: (x + residual) / sqrt(mean square + eps) * weight; in 8 bits a group of channels has as its scale the least power
of two (2^-100 or more) that brings its largest magnitude to 448 or less, and codes are float8_e4m3fn.
Pages: refs int32 [pages] counts the places of the tables that hold a page; tables have -1 where a sequence has none. A place
that the newest rows fall into gets the lowest free page, sequence by sequence and place by place, if it has none or shares its
own (1 < refs); a shared page that holds tokens before those rows is copied. Lengths of a case's sequences follow from its
sizes and "mix" alone.
"""
import math
import random

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
# (query heads, key heads, width)
HEADS = {"16x16x128": (16, 16, 128), "32x4x128": (32, 4, 128), "28x4x128": (28, 4, 128), "16x2x256": (16, 2, 256),
         "32x2x256": (32, 2, 256), "12x4x64": (12, 4, 64), "8x8x64": (8, 8, 64)}
EPS = 1e-6


def listed():
    return [
        # one token's row between two layers: nothing but latency
        dict(name="norm_1_token", kind="norm", T=1, H=2048, heads=0, dtype="bf16", residual=True, group=0),
        # the query heads of a prompt chunk, a part of the product that also gives keys and values
        dict(name="norm_heads_2048", kind="norm", T=2048, H=128, heads=32, dtype="f16", residual=False, group=0),
        # a whole prompt chunk of the residual stream
        dict(name="norm_8192", kind="norm", T=8192, H=4096, heads=0, dtype="bf16", residual=True, group=0),
        # the same rows for a product in 8 bits, or to be sent to other GPUs
        dict(name="norm_codes_8192", kind="norm", T=8192, H=4096, heads=0, dtype="bf16", residual=True, group=128),
        # one step of continuous batching: a few sequences leave, others begin, some write to a page that they share
        dict(name="pages_step_64", kind="step", heads="32x4x128", page=64, pages=16384, seqs=64, longest=8192, mix=21),
        # eight beams, reordered at every token
        dict(name="pages_beam_8", kind="beam", heads="16x2x256", page=64, pages=4096, seqs=8, longest=4001, mix=22),
        # a pool that has become sparse: its pages moved together
        dict(name="pages_compact", kind="compact", heads="32x4x128", page=64, pages=8192, seqs=96, longest=8192, mix=23),
        # a few short chunks of chats: latency
        dict(name="chunk_short", kind="chunk", heads="16x16x128", dtype="bf16", page=64, seqs=4, rows=48, past=900, mix=24),
        # a tree of drafts, or a short message, after a long document: few rows, many keys
        dict(name="chunk_48_long", kind="chunk", heads="32x4x128", dtype="bf16", page=64, seqs=1, rows=48, past=131000, mix=25),
        # chunks of several prompts in one pass, of different lengths, heads in groups of 7
        dict(name="chunk_mixed", kind="chunk", heads="28x4x128", dtype="bf16", page=32, seqs=12, rows=700, past=9000, mix=26),
        # the same with wide heads and float16
        dict(name="chunk_wide", kind="chunk", heads="16x2x256", dtype="f16", page=64, seqs=3, rows=1024, past=8000, mix=27),
        # a late chunk of one long prompt
        dict(name="chunk_2048_long", kind="chunk", heads="32x4x128", dtype="bf16", page=128, seqs=1, rows=2048, past=32768,
             mix=28),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "norm", "step", "beam", "compact", "chunk", "chunk", "chunk", "chunk"])
    mix = rng.randrange(1 << 20)
    if kind == "norm":
        group = rng.choice([0, 0, 32, 128, -1])  # -1: one scale a row
        if rng.random() < 0.3:
            return dict(kind=kind, T=_log_int(rng, 1, 4096), H=rng.choice([64, 128, 256]), heads=rng.choice([1, 4, 12, 32]),
                        dtype=rng.choice(["f16", "bf16"]), residual=False, group=0)
        unit = rng.choice([1, 8]) if group <= 0 else group
        width = max(unit, _log_int(rng, 64, 8192) // unit * unit)
        return dict(kind=kind, T=_log_int(rng, 1, max(1, min(8192, (1 << 25) // width))), H=width, heads=0,
                    dtype=rng.choice(["f16", "bf16", "bf16", "f32"]), residual=rng.random() < 0.7, group=group)
    heads = rng.choice(sorted(HEADS))
    page = rng.choice([32, 64, 128])
    if kind in ("step", "beam", "compact"):
        _, hk, d = HEADS[heads]
        most = (1 << 29) // (hk * d * page)
        seqs = _log_int(rng, 1, 128) if kind != "beam" else _log_int(rng, 2, 32)
        pages = _log_int(rng, 64, min(16384, most))
        return dict(kind=kind, heads=heads, page=page, pages=pages, seqs=seqs, mix=mix,
                    longest=_log_int(rng, 40, min(16384, max(41, pages * page // 2))))
    seqs = rng.choice([1, 1, _log_int(rng, 2, 24)])
    case = dict(kind=kind, heads=heads, dtype=rng.choice(["f16", "bf16"]), page=page, seqs=seqs, rows=_log_int(rng, 17, 4096),
                past=_log_int(rng, 1, 131072 // seqs), mix=mix)
    while work(case)["flops"] > 1.1e12:
        case["rows"] = max(17, case["rows"] * 2 // 3)
        case["past"] = case["past"] * 2 // 3
    return case


# ---- sizes -----------------------------------------------------------------------------------------------------

def _chunks(case):
    """(new rows, tokens before them) of each sequence: one of the most, the others spread below it, over the logarithm; some
    begin with this chunk."""
    rng = random.Random(case["mix"])
    rows = [case["rows"]] + [_log_int(rng, max(1, case["rows"] // 16), case["rows"]) for _ in range(case["seqs"] - 1)]
    past = [case["past"]] + [rng.choice([0, _log_int(rng, max(1, case["past"] // 16), case["past"]),
                                         _log_int(rng, max(1, case["past"] // 4), case["past"])]) for _ in range(case["seqs"] - 1)]
    return rows, past


def _pool(case, seed):
    """A pool's state as lists: refs, table, and the step's lens, rows, keep (and parents). Pages are held all over the pool;
    about a quarter of the sequences go on from one they share their whole pages, and the begun one, with. The seed says which
    pages are held; how many a compaction has to move does not change with it."""
    rng = random.Random(case["mix"])
    pages, page, n = case["pages"], case["page"], case["seqs"]
    free = list(range(pages))
    rng.shuffle(free)
    # half of the pool, about, is to be held
    room = max(n, pages // 2)
    width = -(-(case["longest"] + 2 * page) // page)
    table, lens = [], []
    for b in range(n):
        long = min(case["longest"], max(1, room * page // n))
        at = long if b == 0 else _log_int(rng, max(1, long // 16), long)
        old = rng.randrange(b) if b else 0
        if b and (case["kind"] == "beam" or rng.random() < 0.25) and lens[old] >= page:
            row, at = list(table[old]), lens[old]
            if case["kind"] == "beam":  # beams that went apart some tokens ago
                last = -(-at // page) - 1
                row[last] = free.pop()
        else:
            row = [free.pop() for _ in range(-(-at // page))] if -(-at // page) < len(free) - n else []
            at = at if row else 0
            row = row + [-1] * (width - len(row))
        table.append(row)
        lens.append(at)
    keep, rows, parents = list(lens), [1] * n, [rng.randrange(n) for _ in range(n)]
    now = [x + 1 for x in lens]
    if case["kind"] == "step":
        for b in range(n):
            if rng.random() < 0.1:  # finished; a new prompt begins in its place
                keep[b], rows[b] = 0, _log_int(rng, 1, min(512, case["longest"]))
                now[b] = rows[b]
    if case["kind"] == "beam":
        now = [lens[p] + 1 for p in parents]
    rng = random.Random(seed)
    used = len({p for row in table for p in row if p >= 0})
    low, high = list(range(used)), list(range(used, pages))
    rng.shuffle(low)
    rng.shuffle(high)
    other = low + high + [-1]  # (the last for -1)
    table = [[other[p] for p in row] for row in table]
    refs = [0] * pages
    for row in table:
        for p in row:
            if p >= 0:
                refs[p] += 1
    return refs, table, now, rows, keep, parents


def _page_bytes(case):
    _, hk, d = HEADS[case["heads"]]
    return 2 * hk * d * case["page"]


def work(case):
    if case["kind"] == "norm":
        n, size = case["T"] * case["H"] * max(1, case["heads"]), 2 if case["dtype"] != "f32" else 4
        # x (and the residual) read, the row (and the sum) written; a row of codes comes back in 16 bits
        reads = size * (2 if case["residual"] else 1)
        writes = (2 if case["group"] else size) + (size if case["residual"] else 0)
        return {"bytes": n * (reads + writes), "flops": 4 * n}
    if case["kind"] in ("step", "beam", "compact"):
        width = -(-(case["longest"] + 2 * case["page"]) // case["page"])
        state = 4 * (2 * case["pages"] + 2 * case["seqs"] * width)
        refs, table, now, rows, _, parents = _pool(case, 0)
        if case["kind"] == "compact":
            used = sum(r > 0 for r in refs)
            moved = sum(r > 0 for r in refs[used:])
        elif case["kind"] == "beam":
            moved = sum(1 for p, n in zip(parents, now) if parents.count(p) > 1 and (n - 1) % case["page"])
        else:
            moved = sum(1 for b, n in enumerate(now) if rows[b] == 1 and n > 1 and (n - 1) % case["page"] and
                        refs[table[b][(n - 1) // case["page"]]] > 1)
        # a copied page's codes read and written, and given in 16 bits
        return {"bytes": state + 4 * moved * _page_bytes(case), "flops": 0}
    hq, hk, d = HEADS[case["heads"]]
    rows, past = _chunks(case)
    pairs = sum(r * p + r * (r + 1) // 2 for r, p in zip(rows, past))
    return {"bytes": 2 * (sum(rows) + sum(past)) * hk * d + 4 * sum(rows) * hq * d, "flops": 4 * hq * d * pairs}


# ---- inputs ----------------------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _cu(lengths):
    total, out = 0, [0]
    for n in lengths:
        total += n
        out.append(total)
    return _ints(out)


def _held(gen, n, hk, page, d, spread):
    """n pages of random tokens in the cache's form, and their scales, some hundred pages at a time."""
    codes = torch.empty((n, hk, page, d), dtype=torch.float8_e4m3fn, device="cuda")
    scales = torch.empty((n, hk), dtype=torch.float32, device="cuda")
    for at in range(0, n, 512):
        x = _normal(gen, min(512, n - at), hk, page, d) * spread[:, None, :]
        s = _need(x.abs().amax((2, 3)))
        codes[at:at + 512] = (x / s[..., None, None]).to(torch.float8_e4m3fn)
        scales[at:at + 512] = s
    return codes, scales


def prepare(case, seed):
    gen, s = _gen(seed), dict(case)
    if case["kind"] == "norm":
        t, h, dt = case["T"], case["H"], DTYPES[case["dtype"]]
        # channels that stand out, as the residual stream has them
        spread = torch.exp(_normal(gen, h))
        if case["heads"]:
            whole = _normal(gen, t, 2 * case["heads"], h) * spread
            s["x"] = whole.to(dt)[:, :case["heads"]]
        else:
            s["x"] = (_normal(gen, t, h) * spread).to(dt)
        s["res"] = (4 * _normal(gen, t, h) * spread).to(dt) if case["residual"] else None
        s["w"] = (1 + 0.2 * _normal(gen, h)).to(dt)
        return s
    hq, hk, d = HEADS[case["heads"]]
    page = case["page"]
    spread = torch.exp(0.5 * _normal(gen, hk, d))
    if case["kind"] == "chunk":
        rows, past = _chunks(case)
        lens = [r + p for r, p in zip(rows, past)]
        counts = [-(-n // page) for n in lens]
        n = sum(counts) + 3
        order = torch.randperm(n, generator=gen, device="cuda").to(torch.int32)
        s["table"] = torch.full((len(lens), max(counts)), -1, dtype=torch.int32, device="cuda")
        at = 0
        for b, c in enumerate(counts):
            s["table"][b, :c] = order[at:at + c]
            at += c
        s["lens"], s["cu"], s["longest"] = _ints(lens), _cu(rows), max(lens)
        s["row_list"], s["len_list"] = rows, lens
        s["q"] = _normal(gen, sum(rows), hq, d).to(DTYPES[case["dtype"]])
    else:
        refs, table, now, rows, keep, parents = _pool(case, seed)
        s["refs0"], s["table0"], s["lens"] = _ints(refs), _ints(table), _ints(now)
        s["cu"], s["keep"], s["parents"] = _cu(rows), _ints(keep), _ints(parents)
        s["refs"], s["table"] = s["refs0"].clone(), s["table0"].clone()
        n = case["pages"]
        # how many pages come back: those of the step's copies, or the ones that a compaction moves
        used = sum(r > 0 for r in refs)
        s["back"] = sum(r > 0 for r in refs[used:]) if case["kind"] == "compact" else case["seqs"]
        s["back_cu"] = _ints([page * i for i in range(s["back"] + 1)])
    s["k"], s["k_scale"] = _held(gen, n, hk, page, d, spread)
    s["v"], s["v_scale"] = _held(gen, n, hk, page, d, torch.ones_like(spread))
    return s


# ---- the plain forms -------------------------------------------------------------------------------------------

def _need(most):
    """The least power of two, 2^-100 or more, that brings `most` to 448 or less."""
    m, e = torch.frexp(most)
    e = torch.where(most > 0, e - 9 + (m > 0.875).to(e.dtype), -100).clamp(min=-100)
    return ((e + 127) << 23).view(torch.float32)  # 2^e by its bits


def _plain_norm(s):
    x = s["x"].to(torch.float32)
    if s["res"] is not None:
        x = x + s["res"].to(torch.float32)
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * s["w"].to(torch.float32)
    if s["group"]:
        g = y.unflatten(-1, (-1, s["group"] if s["group"] > 0 else s["H"]))
        scale = _need(g.abs().amax(-1, keepdim=True))
        y = ((g / scale).to(torch.float8_e4m3fn).to(torch.float32) * scale).flatten(-2).to(torch.bfloat16)
    else:
        y = y.to(s["x"].dtype)
    return y if s["res"] is None else (y, x.to(s["x"].dtype))


def _count(refs, table, by):
    """refs with `by` added for every place of the table that holds a page."""
    there = (table >= 0) & (table < refs.numel())
    at = torch.where(there, table, 0).flatten().long()
    return refs.index_add(0, at, torch.where(there, by, 0).flatten().to(torch.int32))


def _plain_take(refs, table, lens, cu, page):
    """(refs, table, src, dst, short) after the newest rows' places have pages of their own."""
    rows = cu[1:] - cu[:-1]
    first = (lens - rows).clamp(min=0) // page
    place = torch.arange(table.shape[1], device="cuda")
    fallen = (place >= first[:, None]) & (place * page < lens[:, None]) & (rows > 0)[:, None]
    there = (table >= 0) & (table < refs.numel())
    shared = there & (refs[torch.where(there, table, 0).long()] > 1)
    needs = fallen & (shared | ~there)
    # the lowest free pages, in the order of the places that need one
    free = refs == 0
    order = torch.argsort(free.logical_not().to(torch.uint8), stable=True).to(torch.int32)
    rank = torch.cumsum(needs.flatten(), 0).view_as(table) - 1
    found = needs & (rank < free.sum())
    given = torch.where(found, order[rank.clamp(0, refs.numel() - 1)], -1)
    copied = found & shared & (place == first[:, None]) & ((lens - rows) % page > 0)[:, None]
    src = torch.where(copied, table, -1).amax(1)
    dst = torch.where(copied, given, -1).amax(1)
    refs = _count(refs, torch.where(needs & shared, table, -1), -1)
    refs = _count(refs, torch.where(found, given, -1), 1)
    return refs, torch.where(needs, given, table), src, dst, (needs & ~found).sum(1).to(torch.int32)


def _plain_copies(s, src, dst):
    there = dst >= 0
    # in the place of a pair that is not there, the first one that is (page 0 onto itself where there is none)
    first = torch.argmax(there.to(torch.uint8))
    a, b = (torch.where(there, x, torch.where(there[first], x[first], 0)).long() for x in (src, dst))
    for codes, scales in ((s["k"], s["k_scale"]), (s["v"], s["v_scale"])):
        raw = codes.view(torch.uint8)
        for i in range(0, a.numel(), 4096):
            raw[b[i:i + 4096]] = raw[a[i:i + 4096]]
            scales[b[i:i + 4096]] = scales[a[i:i + 4096]]


def _plain_back(s, dst):
    """(k, v): the tokens of the pages dst in bfloat16, zeros where there is none."""
    dst, out = dst[:s["back"]], []
    at = dst.clamp(min=0).long()
    for codes, scales in ((s["k"], s["k_scale"]), (s["v"], s["v_scale"])):
        x = codes.view(torch.uint8)[at].view(torch.float8_e4m3fn).to(torch.float32) * scales[at][..., None, None]
        x = torch.where((dst >= 0)[:, None, None, None], x, 0.0)
        out.append(x.transpose(1, 2).flatten(0, 1).to(torch.bfloat16))
    return out


def _plain_pages(s):
    refs, table, page = s["refs0"], s["table0"], s["page"]
    if s["kind"] == "compact":
        n = refs.numel()
        held, number = refs > 0, torch.arange(n, dtype=torch.int32, device="cuda")
        used = held.sum().to(torch.int32)
        leaves, takes = held & (number >= used), ~held & (number < used)
        # the held pages past the first `used` numbers go to the free ones among those, both in order
        half = max(1, n // 2)
        src = torch.argsort(leaves.logical_not().to(torch.uint8), stable=True).to(torch.int32)[:half]
        dst = torch.argsort(takes.logical_not().to(torch.uint8), stable=True).to(torch.int32)[:half]
        there = torch.arange(half, device="cuda") < leaves.sum()
        goes = torch.where(there, src, 0).long()
        to = number.index_add(0, goes, torch.where(there, dst - src, 0))
        refs = torch.where(leaves, 0, refs).index_add(0, torch.where(there, dst, 0).long(), torch.where(there, refs[goes], 0))
        table = torch.where((table >= 0) & (table < n), to[table.clamp(0, n - 1).long()], table)
        src, dst = torch.where(there, src, -1), torch.where(there, dst, -1)
        _plain_copies(s, src, dst)
        return (table, refs, src, dst, used.view(1), *_plain_back(s, dst))
    if s["kind"] == "beam":
        old, parents = table, s["parents"].long()
        table = old[parents]
        refs = _count(_count(refs, old, -1), table, 1)
    else:
        gone = torch.arange(table.shape[1], device="cuda") * page >= s["keep"][:, None]
        refs = _count(refs, torch.where(gone, table, -1), -1)
        table = torch.where(gone, -1, table)
    refs, table, src, dst, short = _plain_take(refs, table, s["lens"], s["cu"], page)
    _plain_copies(s, src, dst)
    return (table, refs, src, dst, short, *_plain_back(s, dst))


def _plain_chunk(s):
    hq, hk, d = HEADS[s["heads"]]
    g, out, at = hq // hk, torch.empty_like(s["q"]), 0
    for b, (r, n) in enumerate(zip(s["row_list"], s["len_list"])):
        pages = s["table"][b, :-(-n // s["page"])].long()
        k, v = ((c.view(torch.uint8)[pages].view(torch.float8_e4m3fn).to(torch.float32) * e[pages][..., None, None])
                .transpose(0, 1).flatten(1, 2)[:, :n] for c, e in ((s["k"], s["k_scale"]), (s["v"], s["v_scale"])))
        q = s["q"][at:at + r].to(torch.float32).view(r, hk, g, d).permute(1, 2, 0, 3).reshape(hk, g * r, d)
        seen = torch.arange(n, device="cuda") <= torch.arange(n - r, n, device="cuda")[:, None]
        scores = (q @ k.transpose(1, 2)).view(hk, g, r, n).mul_(d ** -0.5).masked_fill_(~seen, float("-inf"))
        scores.sub_(scores.amax(-1, keepdim=True)).exp_()
        o = (scores.view(hk, g * r, n) @ v).view(hk, g, r, d) / scores.sum(-1, keepdim=True)
        out[at:at + r] = o.permute(2, 0, 1, 3).reshape(r, hq, d).to(out.dtype)
        at += r
    return out


# ---- one pass --------------------------------------------------------------------------------------------------

def _own(s):
    from larder_amd import attention, pages, trunk
    if s["kind"] == "norm":
        if not s["group"]:
            return trunk.norm_rows(s["x"], s["w"], EPS, residual=s["res"])
        got = trunk.norm_rows(s["x"], s["w"], EPS, residual=s["res"], group=s["group"] if s["group"] > 0 else s["H"])
        y = trunk.read_codes(got[0], got[1], dtype=torch.bfloat16)
        return y if s["res"] is None else (y, got[2])
    cache = attention.KVCache(s["k"], s["k_scale"], s["v"], s["v_scale"])
    if s["kind"] == "chunk":
        return attention.chunk_rows(s["q"], cache, s["table"], s["lens"], s["cu"], longest=s["longest"])
    refs, table, page = s["refs"].copy_(s["refs0"]), s["table"].copy_(s["table0"]), s["page"]
    if s["kind"] == "compact":
        src, dst, tail = pages.compact_pages(refs, table)
    else:
        if s["kind"] == "beam":
            table = pages.fork_pages(refs, table, s["parents"])
        else:
            pages.free_pages(refs, table, s["keep"], page=page)
        src, dst, tail = pages.take_pages(refs, table, s["lens"], s["cu"], page=page)
    pages.copy_pages(cache, src, dst)
    k, v = attention.read_rows(cache, dst[:s["back"]].view(-1, 1), s["back_cu"], s["back"] * page)
    return table, refs, src, dst, tail, k, v


def run(state):
    if own:
        return _own(state)
    return {"norm": _plain_norm, "chunk": _plain_chunk}.get(state["kind"], _plain_pages)(state)


# ---- the answers in 64 bits ------------------------------------------------------------------------------------

def _exact_codes(x):
    """x rounded to the nearest e4m3 value (ties to even), as float64; |x| <= 448."""
    e = torch.clamp(torch.frexp(x)[1] - 1, min=-6) - 3
    step = ((e.to(torch.int64) + 1023) << 52).view(torch.float64)
    return torch.round(x / step) * step


def _exact_norm(s):
    total = s["x"].to(torch.float64)
    if s["res"] is not None:
        total = total + s["res"].to(torch.float64)
    length = torch.linalg.vector_norm(total, dim=-1, keepdim=True)
    y = total * s["w"].to(torch.float64) * torch.rsqrt(length.square() / s["H"] + EPS)
    if s["group"]:
        parts = torch.stack(y.split(s["group"] if s["group"] > 0 else s["H"], -1), -2)
        m, e = torch.frexp((parts.abs().amax(-1, keepdim=True) / 448).clamp(min=2.0 ** -100))
        scale = (((e - (m == 0.5).to(e.dtype)).to(torch.int64) + 1023) << 52).view(torch.float64)
        y = (_exact_codes(parts / scale) * scale).reshape(y.shape)
    return y if s["res"] is None else (y, total)


def _exact_pages(s):
    refs, table, page = s["refs0"].tolist(), s["table0"].tolist(), s["page"]
    if s["kind"] == "compact":
        used = len(refs) - refs.count(0)
        src = [p for p in range(used, len(refs)) if refs[p]]
        dst = [p for p in range(used) if not refs[p]]
        to = dict(zip(src, dst))
        for a, b in to.items():
            refs[a], refs[b] = 0, refs[a]
        table = [[to.get(p, p) for p in row] for row in table]
        pad = [-1] * (max(1, len(refs) // 2) - len(src))
        src, dst, tail = src + pad, dst + pad, [used]
    else:
        if s["kind"] == "beam":
            new = [list(table[p]) for p in s["parents"].tolist()]
        else:
            new = [[p if i < -(-k // page) else -1 for i, p in enumerate(row)] for row, k in zip(table, s["keep"].tolist())]
        refs = [0] * len(refs)
        for row in new:
            for p in row:
                if p >= 0:
                    refs[p] += 1
        table, before = [list(row) for row in new], list(refs)
        free = iter([p for p, r in enumerate(refs) if r == 0])
        src, dst, tail, cu = [], [], [], s["cu"].tolist()
        for b, n in enumerate(s["lens"].tolist()):
            start, a, c, missing = n - (cu[b + 1] - cu[b]), -1, -1, 0
            for i in range(start // page, -(-n // page)):
                p = table[b][i]
                if p >= 0 and before[p] == 1:
                    continue
                got = next(free, -1)
                missing += got < 0
                if got >= 0:
                    refs[got] += 1
                if p >= 0:
                    refs[p] -= 1
                    if got >= 0 and i * page < start:
                        a, c = p, got
                table[b][i] = got
            src.append(a)
            dst.append(c)
            tail.append(missing)
    back = []
    for codes, scales in ((s["k"], s["k_scale"]), (s["v"], s["v_scale"])):
        raw, scales, out = codes.view(torch.uint8), scales.to(torch.float64), []
        for at in range(0, s["back"], 256):
            some = _ints(src[at:at + 256][:s["back"] - at]).long()
            x = raw[some.clamp(min=0)].view(torch.float8_e4m3fn).to(torch.float64) * scales[some.clamp(min=0)][..., None, None]
            x[some < 0] = 0.0
            out.append(x.transpose(1, 2).flatten(0, 1))
        back.append(torch.cat(out) if out else torch.zeros((0, codes.shape[1], codes.shape[3]), dtype=torch.float64, device="cuda"))
    return (_ints(table), _ints(refs), _ints(src), _ints(dst), _ints(tail), *back)


def _exact_chunk(s):
    hq, hk, d = HEADS[s["heads"]]
    page, cu, out = s["page"], s["cu"].tolist(), []
    for b, n in enumerate(s["lens"].tolist()):
        pages = s["table"][b, :-(-n // page)].long()
        k, v = ((c.view(torch.uint8)[pages].view(torch.float8_e4m3fn).to(torch.float64) * e[pages][..., None, None])
                .transpose(1, 2).flatten(0, 1)[:n] for c, e in ((s["k"], s["k_scale"]), (s["v"], s["v_scale"])))
        q = s["q"][cu[b]:cu[b + 1]].to(torch.float64)
        o = torch.empty_like(q)
        hidden = torch.arange(n, device="cuda") > torch.arange(q.shape[0], device="cuda")[:, None] + n - q.shape[0]
        for h in range(hq):
            x = (q[:, h] @ k[:, h * hk // hq].t()) / math.sqrt(d)
            o[:, h] = torch.softmax(x.masked_fill(hidden, float("-inf")), -1) @ v[:, h * hk // hq]
        out.append(o)
    return torch.cat(out)


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "chunk": _exact_chunk}.get(case["kind"], _exact_pages)(s)
