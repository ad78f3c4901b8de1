"""Rotary positions, the paged 8-bit cache and attention in float64 numpy, from their definitions: what the kernels of
larder_amd.attention are held to. Rows are packed [T, heads, width]; cu [B + 1] says where each sequence begins."""
import numpy as np

__all__ = ["E4M3", "append", "attend", "encode_e4m3", "read", "restate", "rope", "scale_for", "softmax_rows"]


def _e4m3_values():
    v = np.empty(256)
    for c in range(256):
        sign, e, m = -1.0 if c & 0x80 else 1.0, (c >> 3) & 15, c & 7
        v[c] = np.nan if c & 0x7f == 0x7f else sign * (m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7))
    return v


E4M3 = _e4m3_values()
_POSITIVE = E4M3[:0x7f]


def encode_e4m3(x):
    """uint8 codes of float64 values within 448, to the nearest, ties to the even code; NaN and infinities to NaN."""
    x = np.asarray(x, np.float64)
    mag = np.where(np.isfinite(x), np.abs(x), 0.0)
    hi = np.clip(np.searchsorted(_POSITIVE, mag), 1, len(_POSITIVE) - 1)
    lo = hi - 1
    mid = (_POSITIVE[lo] + _POSITIVE[hi]) / 2
    code = np.where((mag > mid) | ((mag == mid) & (hi % 2 == 0)), hi, lo).astype(np.uint8)
    code = code | (np.signbit(x).astype(np.uint8) << 7)
    return np.where(np.isfinite(x), code, np.uint8(0x7f)).astype(np.uint8)


def scale_for(most):
    """The least power of two, 2^-100 or more, that brings `most` to 448 or less."""
    m, e = np.frexp(np.asarray(most, np.float64) / 448)
    s = np.where(m == 0.5, e - 1, e)
    return np.ldexp(1.0, np.where(np.asarray(most) > 0, np.maximum(s, -100), -100))


def rope(x, positions, freq, interleaved=False, gain=1.0):
    x = np.array(x, np.float64)
    f = len(freq)
    a = np.asarray(positions, np.float64)[:, None, None] * np.asarray(freq, np.float64)
    c, s = gain * np.cos(a), gain * np.sin(a)
    u, w = (x[..., 0:2 * f:2], x[..., 1:2 * f:2]) if interleaved else (x[..., :f], x[..., f:2 * f])
    p, q = u * c - w * s, w * c + u * s
    if interleaved:
        x[..., 0:2 * f:2], x[..., 1:2 * f:2] = p, q
    else:
        x[..., :f], x[..., f:2 * f] = p, q
    return x


def restate(codes, ratio):
    return encode_e4m3(E4M3[codes] * ratio)


def append(codes, scales, rows, cu, lens, table):
    """rows [T, heads, width] float64 into codes [pages, heads, page, width] uint8 and scales [pages, heads], in place."""
    pages, heads, page, _ = codes.shape
    for b, n in enumerate(lens):
        start = n - (cu[b + 1] - cu[b])
        if cu[b + 1] == cu[b]:
            continue
        for p in range(max(start, 0) // page, -(-n // page)):
            lo, hi = max(start, p * page), min(n, (p + 1) * page)
            if hi <= lo or p >= table.shape[1] or not 0 <= table[b, p] < pages:
                continue
            at, x = table[b, p], rows[cu[b] + lo - start:cu[b] + hi - start]
            for h in range(heads):
                y = x[:, h]
                need = scale_for(np.max(np.where(np.isfinite(y), np.abs(y), 0.0)))
                held = lo - p * page
                old = scales[at, h] if held else 0.0
                now = max(old, need)
                if held and now != old:
                    codes[at, h, :held] = restate(codes[at, h, :held], old / now)
                codes[at, h, held:held + hi - lo] = encode_e4m3(y / now)
                scales[at, h] = now


def read(codes, scales, table_row, n):
    """(values [n, heads, width] float64, there [n] bool): a sequence's first n tokens; those of no page are zero."""
    pages, heads, page, width = codes.shape
    out, there = np.zeros((n, heads, width)), np.zeros(n, bool)
    for t in range(n):
        p = t // page
        if p < len(table_row) and 0 <= table_row[p] < pages:
            at = table_row[p]
            out[t] = E4M3[codes[at, :, t % page]] * scales[at][:, None]
            there[t] = True
    return out, there


def softmax_rows(x, seen):
    """Weights over the last axis where seen; all zero where nothing is."""
    x = np.where(seen, x, -np.inf)
    m = np.max(x, -1, keepdims=True, initial=-np.inf)
    m = np.where(np.isneginf(m), 0.0, m)
    with np.errstate(invalid="ignore"):
        e = np.where(seen, np.exp(x - m), 0.0)
    s = e.sum(-1, keepdims=True)
    return np.divide(e, s, out=np.zeros_like(e), where=s != 0)


def attend(q, k, v, scale, there=None):
    """q [n, q_heads, width] over k, v [m, heads, width] float64, aligned at their ends: row i sees keys j <= i + m - n (that are
    `there`). Returns (out, spread): spread [n, q_heads, width] = sum p |v|, which bounds what rounding weights can do; values
    that a row does not see play no part, whatever they are."""
    n, hq, _ = q.shape
    m, hk, _ = k.shape
    seen = np.arange(m) <= np.arange(n)[:, None] + (m - n)
    if there is not None:
        seen = seen & there
    out, spread = np.zeros(q.shape), np.zeros(q.shape)
    with np.errstate(invalid="ignore"):
        for h in range(hq):
            g = h // (hq // hk)
            p = softmax_rows(q[:, h] @ k[:, g].T * scale, seen)
            for i in range(n):
                j = seen[i]
                out[i, h], spread[i, h] = p[i, j] @ v[j, g], p[i, j] @ np.abs(v[j, g])
    return out, spread
