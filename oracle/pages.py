"""The pages of the paged cache as a pool that tables share, from its definition in plain Python: what larder_amd.pages is held
to. refs is a list, tables lists of lists; every function returns new ones."""

__all__ = ["compact", "fork", "free", "take"]


def _held(p, refs):
    return 0 <= p < len(refs)


def take(refs, table, lens, cu, page):
    """(refs, table, src, dst, lacking) after each place that the newest rows fall into has a page of its own."""
    refs, table, before = list(refs), [list(row) for row in table], list(refs)
    free = iter([p for p, r in enumerate(before) if r == 0])
    src, dst, lacking = [-1] * len(table), [-1] * len(table), [0] * len(table)
    for b, n in enumerate(lens):
        rows = 1 if cu is None else cu[b + 1] - cu[b]
        if rows <= 0 or n <= 0:
            continue
        start = max(n - rows, 0)
        for i in range(start // page, min(-(-n // page), len(table[b]))):
            old = table[b][i]
            if _held(old, refs) and before[old] <= 1:
                continue
            new = next(free, -1)
            if new < 0 and _held(old, refs) and refs[old] == 1:
                continue  # the others have given it up: it is this sequence's own
            table[b][i] = new
            if new >= 0:
                refs[new] = 1
            else:
                lacking[b] += 1
            if _held(old, refs):
                refs[old] -= 1
                if new >= 0 and start > i * page:
                    src[b], dst[b] = old, new
    return refs, table, src, dst, lacking


def free(refs, table, keep, page):
    refs, out = list(refs), []
    for row, k in zip(table, keep):
        n = -(-max(k, 0) // page)
        for p in row[n:]:
            if _held(p, refs):
                refs[p] -= 1
        out.append(row[:n] + [-1] * len(row[n:]))
    return refs, out


def fork(refs, table, parents):
    refs, width = list(refs), len(table[0])
    new = [list(table[p]) if 0 <= p < len(table) else [-1] * width for p in parents]
    new = [[p if _held(p, refs) else -1 for p in row] for row in new]
    for rows, by in ((table, -1), (new, 1)):
        for row in rows:
            for p in row:
                if _held(p, refs):
                    refs[p] += by
    return refs, new


def compact(refs, tables):
    """(refs, tables, src, dst, used): the held pages past the first `used` numbers to the free ones among those, in order."""
    used = sum(r > 0 for r in refs)
    src = [p for p in range(used, len(refs)) if refs[p] > 0]
    dst = [p for p in range(used) if refs[p] <= 0]
    to, out = dict(zip(src, dst)), list(refs)
    for a, b in to.items():
        out[b], out[a] = refs[a], 0
    return out, [[[to.get(p, p) for p in row] for row in t] for t in tables], src, dst, used
