"""Attention of the trunk's rows on MI355X: rotary positions, a paged 8-bit key / value cache, attention of single tokens
over it and of whole prompts. Inference only; every call queues its kernels on the current stream and none waits for the
GPU.

    rotary_freq(width, base, kind, factor, ...)   -> (freq, gain): what rope_rows and append_rows rotate by
    rope_rows(x, positions, freq, ...)            x with each head rotated by its row's position (route_cuda.py:549-591)
    KVCache, KVCache.empty(pages, heads, width)   the cache's four tensors
    append_rows(cache, q, k, v, table, lens, ...) rotates q and k and writes the rows' keys and values into their pages
    read_rows(cache, table, cu, total)            the first tokens of each sequence back in 16 (or 32) bits
    attend_rows(q, cache, table, lens, ...)       the newest rows of each sequence over its cached tokens
    prompt_rows(q, k, v, cu, ...)                 packed sequences, causal, over their own keys and values

Rows are packed: tensors [T, heads, width] hold the sequences one after the other, and cu int32 [sequences + 1] says where
each begins (cu[0] = 0; one row a sequence where cu is None). Rows of no sequence come back zero. Heads are 64, 128 or 256
channels wide, and any number of query heads shares a key head. Rows may be strided views, as of a product that gives q, k
and v side by side; one whose layout no kernel reads is copied first.

lens int32 [sequences] counts a sequence's tokens with the rows of the call among them: row r of n stands at place lens -
n + r. table int32 [sequences, width] lists each sequence's pages in order; entries behind its last page are not read. A
page outside the cache (or the table) holds nothing: no token is written there and none is seen. Sequences may share pages
they only read; a page that a call writes to belongs to one of them.
"""
import math
from typing import NamedTuple

import torch

from . import _lib
from ._lib import call, dcode, stream

__all__ = ["KVCache", "append_rows", "attend_rows", "prompt_rows", "read_rows", "rope_rows", "rotary_freq"]


class KVCache(NamedTuple):
    """e4m3 codes [pages, heads, page, width] of keys and of values, and one float32 scale for each page and head of either.

    A scale is the least power of two (2^-100 at least) that brings the page's largest finite magnitude to 448 or less; a
    page that held tokens keeps the larger of its old and the new scale, its codes restated in that (exactly, unless they
    become subnormal). Infinities and NaN are kept as NaN. A page's old contents count for nothing once a sequence begins it
    anew, so pages need no clearing."""
    k: torch.Tensor
    k_scale: torch.Tensor
    v: torch.Tensor
    v_scale: torch.Tensor

    @classmethod
    def empty(cls, pages, heads, width, page=64, device="cuda"):
        """A cache of `pages` pages of `page` (32, 64 or 128) tokens."""
        if page not in (32, 64, 128) or width not in (64, 128, 256):
            raise ValueError("KVCache: pages of 32, 64 or 128 tokens, heads of 64, 128 or 256 channels")
        codes = [torch.zeros((pages, heads, page, width), dtype=torch.float8_e4m3fn, device=device) for _ in range(2)]
        scales = [torch.full((pages, heads), 2.0 ** -100, dtype=torch.float32, device=device) for _ in range(2)]
        return cls(codes[0], scales[0], codes[1], scales[1])

    def nbytes(self):
        return sum(t.numel() * t.element_size() for t in self)


def rotary_freq(width, base=10000.0, kind="default", factor=1.0, original=None, beta=(32.0, 1.0), device="cuda"):
    """(freq float64 [width / 2] on the device, gain): the angle a position of each pair of the first `width` channels of a
    head, base^(-2 i / width), stretched for contexts `factor` times as long as the model was trained on:

      "default"  as they are
      "linear"   positions interpolated: every angle divided by factor
      "ntk"      the base raised to base factor^(width / (width - 2)): the slowest pair is interpolated, the fastest kept
      "yarn"     pairs that turn more than beta[0] times in `original` positions kept, those that turn less than beta[1]
                 times interpolated, a ramp between them; gain 0.1 ln(factor) + 1 (the YaRN method)
    """
    if width <= 0 or width % 2:
        raise ValueError("rotary_freq: an even number of channels")
    if factor < 1.0:
        raise ValueError("rotary_freq: a factor of at least 1")
    i = torch.arange(0, width, 2, dtype=torch.float64)
    gain = 1.0
    if kind == "ntk":
        base = base * factor ** (width / (width - 2)) if width > 2 else base
    freq = float(base) ** (-i / width)
    if kind == "linear":
        freq = freq / factor
    elif kind == "yarn":
        if not original:
            raise ValueError("rotary_freq: yarn needs the original context length")

        def pair_of(turns):  # the pair (a real number) that turns so many times in `original` positions
            return width * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))
        low, high = max(math.floor(pair_of(beta[0])), 0), min(math.ceil(pair_of(beta[1])), width // 2 - 1)
        keep = 1.0 - ((torch.arange(width // 2, dtype=torch.float64) - low) / max(high - low, 1e-3)).clamp(0, 1)
        freq = freq * keep + freq / factor * (1.0 - keep)
        gain = 0.1 * math.log(factor) + 1.0
    elif kind not in ("default", "ntk"):
        raise ValueError(f"rotary_freq: {kind!r} is not default, linear, ntk or yarn")
    return freq.to(device), gain


# ---- arguments -------------------------------------------------------------------------------------------------

def _p(t):
    return None if t is None else t.data_ptr()


def _check(fn, ok, why):
    if not ok:
        raise ValueError(f"{fn}: {why}")


def _same_device(fn, first, *others):
    dev = first.device
    _check(fn, first.is_cuda, "tensors must live on the GPU")
    for t in others:
        _check(fn, t is None or t.device == dev, "tensors on different devices")
    return dev


def _rows(fn, name, x, heads=None, width=None, rows=None):
    """A [T, heads, width] tensor the kernels can read (its last axis dense, 16-byte aligned rows), copied if it is not."""
    _check(fn, x.dim() == 3, f"{name} is [rows, heads, width]")
    _check(fn, (heads is None or x.shape[1] == heads) and (width is None or x.shape[2] == width)
           and (rows is None or x.shape[0] == rows), f"{name} is {tuple(x.shape)}")
    st, size = x.stride(), x.element_size()
    if st[2] != 1 or (st[0] * size) % 16 or (st[1] * size) % 16 or x.data_ptr() % 16:
        x = x.contiguous()
        if x.data_ptr() % 16:
            x = x.clone()
    return x


def _ints(fn, name, t, *shape):
    _check(fn, t.dtype == torch.int32 and t.dim() == len(shape) and all(s is None or s == d for s, d in zip(shape, t.shape)),
           f"{name} is int32 {list(shape)}, not {t.dtype} {list(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


def _sequences(fn, cu, lens, table, rows):
    """(cu, lens, table, sequences) checked; lens may be None (read_rows)."""
    n = table.shape[0] if table.dim() == 2 else -1
    table = _ints(fn, "table", table, n, None)
    _check(fn, table.shape[1] > 0, "a table without pages")
    if lens is not None:
        lens = _ints(fn, "lens", lens, n)
    if cu is None:
        _check(fn, rows == n, f"{rows} rows of {n} sequences need their offsets cu")
    else:
        cu = _ints(fn, "cu", cu, n + 1)
    return cu, lens, table, n


def _cache(fn, cache):
    k, ks, v, vs = cache
    _check(fn, k.dim() == 4 and k.dtype in (torch.float8_e4m3fn, torch.uint8) and v.dtype == k.dtype and v.shape == k.shape,
           "the cache's codes are float8_e4m3fn [pages, heads, page, width]")
    _check(fn, ks.dtype == torch.float32 and vs.dtype == torch.float32 and ks.shape == k.shape[:2] and vs.shape == k.shape[:2],
           "the cache's scales are float32 [pages, heads]")
    _check(fn, k.is_contiguous() and v.is_contiguous() and ks.is_contiguous() and vs.is_contiguous(),
           "the cache's tensors must be contiguous")
    return k.shape


def _freq(fn, freq, width):
    if freq is None:
        return None, 0
    _check(fn, freq.dtype == torch.float64 and freq.dim() == 1 and 2 * freq.numel() <= width,
           "freq is float64 [pairs], two channels a pair")
    return freq if freq.is_contiguous() else freq.contiguous(), freq.numel()


def _on(dev, go):
    """go(stream) with dev as the current device."""
    if dev.index == torch.cuda.current_device():
        return go(stream())
    with torch.cuda.device(dev):
        return go(stream())


# ---- the calls -------------------------------------------------------------------------------------------------

def rope_rows(x, positions, freq, interleaved=False, gain=1.0, out=None):
    """x [T, heads, width] (float16, bfloat16 or float32) with the first 2 len(freq) channels of every head rotated by the
    angles positions[t] * freq (positions int32 or int64 [T], any; freq float64, radians): pairs (i, i + len(freq)), or
    (2 i, 2 i + 1) where interleaved, multiplied by gain; the other channels as they are. float32 inside, one rounding.
    out: a tensor of x's shape and type, which may be x; rows of any strides with a dense last axis."""
    fn = "rope_rows"
    _check(fn, x.dim() == 3, "x is [rows, heads, width]")
    t, heads, width = x.shape
    dt = dcode(x.dtype)
    _check(fn, positions.dim() == 1 and positions.shape[0] == t and positions.dtype in (torch.int32, torch.int64),
           "positions is int32 or int64 [rows]")
    freq, pairs = _freq(fn, freq, width)
    _check(fn, freq is not None, "no frequencies")
    if out is None:
        out = torch.empty((t, heads, width), dtype=x.dtype, device=x.device)
    _check(fn, out.shape == x.shape and out.dtype == x.dtype and (width == 1 or out.stride(2) == 1),
           "out has x's shape and type and a dense last axis")
    dev = _same_device(fn, x, positions, freq, out)
    if x.stride(2) != 1 and width > 1:
        x = x.contiguous()
    positions = positions if positions.is_contiguous() else positions.contiguous()
    if x.numel() == 0:
        return out
    _on(dev, lambda st: call("lmoe_rope_rows", _p(x), dt, x.stride(0), x.stride(1), _p(positions),
                             int(positions.dtype == torch.int64), _p(freq), pairs, t, heads, width, int(bool(interleaved)),
                             float(gain), _p(out), out.stride(0), out.stride(1), st))
    return out


def append_rows(cache, q, k, v, table, lens, cu=None, freq=None, interleaved=False, gain=1.0, keys=False):
    """Writes the rows k, v [T, heads, width] of each sequence into its pages, k rotated by the rows' places as rope_rows does
    (freq None: as it is), and returns (q, k): q [T, query heads, width] rotated likewise (None for None), and with keys=True
    the rotated k in its own type, as prompt_rows reads it (else None). float16, bfloat16 or float32. len(freq) is a multiple
    of 8 (of 4 where interleaved). The cache's tensors are written in place."""
    fn = "append_rows"
    pages, heads, page, width = _cache(fn, cache)
    t = k.shape[0]
    k, v = _rows(fn, "k", k, heads, width), _rows(fn, "v", v, heads, width, t)
    _check(fn, v.dtype == k.dtype and (q is None or q.dtype == k.dtype), "q, k and v have one type")
    if q is not None:
        q = _rows(fn, "q", q, None, width, t)
    dt = dcode(k.dtype)
    cu, lens, table, n = _sequences(fn, cu, lens, table, t)
    freq, pairs = _freq(fn, freq, width)
    dev = _same_device(fn, k, v, q, table, lens, cu, freq, *cache)
    q_out = q
    if q is not None and pairs:
        q_out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    turned = q if pairs else None
    k_out = torch.empty(k.shape, dtype=k.dtype, device=dev) if keys else None
    if t and n:
        qs = turned.stride() if turned is not None else (0, 0)
        _on(dev, lambda st: call(
            "lmoe_kv_append", _p(turned), qs[0], qs[1], q.shape[1] if q is not None else 0, _p(k), k.stride(0), k.stride(1),
            _p(v), v.stride(0), v.stride(1), dt, t, heads, width, _p(cu), _p(lens), n, _p(table), table.shape[1],
            _p(cache[0]), _p(cache[1]), _p(cache[2]), _p(cache[3]), pages, page, _p(freq), pairs, int(bool(interleaved)),
            float(gain), _p(q_out) if turned is not None else None, _p(k_out), st))
    elif t:
        q_out = q_out if turned is None else q_out.zero_()
        k_out = k_out if k_out is None else k_out.zero_()
    return q_out, k_out


def read_rows(cache, table, cu, total, dtype=torch.bfloat16):
    """(k, v) [total, heads, width] in dtype: the first cu[b + 1] - cu[b] tokens of every sequence, codes times scale, rounded
    once (bfloat16 holds them exactly): the history that the rows of a later prompt chunk see, for prompt_rows."""
    fn = "read_rows"
    pages, heads, page, width = _cache(fn, cache)
    dt = dcode(dtype)
    _check(fn, cu is not None, "no offsets cu")
    cu, _, table, n = _sequences(fn, cu, None, table, total)
    dev = _same_device(fn, cache[0], *cache[1:], table, cu)
    k, v = (torch.empty((total, heads, width), dtype=dtype, device=dev) for _ in range(2))
    if total:
        _on(dev, lambda st: call("lmoe_kv_read", _p(cache[0]), _p(cache[1]), _p(cache[2]), _p(cache[3]), pages, page, heads,
                                 width, _p(table), table.shape[1], _p(cu), n, total, _p(k), _p(v), dt, st))
    return k, v


def attend_rows(q, cache, table, lens, cu=None, most_rows=None, longest=None, scale=None):
    """softmax(scale q k^T) v of the newest rows q [T, query heads, width] (float16 or bfloat16) over the cached tokens of
    their sequences: row r of a sequence's n sees its first lens - n + r + 1 tokens (a row that sees none is zero); scale is
    width^-0.5 if None. Made for few rows a sequence: one token of each, or a speculative decoder's draft.

    most_rows and longest size the launch: about the most rows of a sequence (1 without cu, else T / sequences) and tokens of
    one (the table's room). Any values give the same sums in another order."""
    fn = "attend_rows"
    pages, heads, page, width = _cache(fn, cache)
    q = _rows(fn, "q", q, None, width)
    t, q_heads = q.shape[0], q.shape[1]
    _check(fn, q.dtype in (torch.float16, torch.bfloat16), f"q is float16 or bfloat16, not {q.dtype}")
    _check(fn, q_heads > 0 and q_heads % heads == 0, f"{q_heads} query heads over {heads} key heads")
    cu, lens, table, n = _sequences(fn, cu, lens, table, t)
    dev = _same_device(fn, q, table, lens, cu, *cache)
    out = torch.empty((t, q_heads, width), dtype=q.dtype, device=dev)
    if not t or not n:
        return out.zero_()
    most = int(most_rows) if most_rows is not None else 1 if cu is None else -(-t // n)
    room = table.shape[1] * page
    long = min(int(longest), room) if longest is not None else room
    need = _lib.lib().lmoe_kv_attend_workspace_bytes(t, q_heads, heads, width, n, max(most, 1), max(long, 1))
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    _on(dev, lambda st: call(
        "lmoe_kv_attend", _p(q), dcode(q.dtype), q.stride(0), q.stride(1), t, q_heads, heads, width, _p(cu), _p(lens), n,
        _p(table), table.shape[1], _p(cache[0]), _p(cache[1]), _p(cache[2]), _p(cache[3]), pages, page, max(most, 1),
        max(long, 1), float(width ** -0.5 if scale is None else scale), _p(ws), need, _p(out), st))
    return out


def prompt_rows(q, k, v, cu, cu_k=None, scale=None):
    """softmax(scale q k^T) v of packed sequences, causal: q [T, query heads, width], k and v [U, heads, width] (float16 or
    bfloat16), sequence b's rows cu[b] .. cu[b + 1] of q and cu_k[b] .. cu_k[b + 1] of k and v (cu_k None: the same rows).
    The last row sees all of its sequence's keys, each row before it one fewer; a row that sees none is zero. scale is
    width^-0.5 if None."""
    fn = "prompt_rows"
    q = _rows(fn, "q", q)
    t, q_heads, width = q.shape
    k = _rows(fn, "k", k, None, width)
    u, heads = k.shape[0], k.shape[1]
    v = _rows(fn, "v", v, heads, width, u)
    _check(fn, q.dtype in (torch.float16, torch.bfloat16) and k.dtype == q.dtype and v.dtype == q.dtype,
           "q, k and v are all float16 or all bfloat16")
    _check(fn, width in (64, 128, 256), f"heads of {width} channels (64, 128 and 256 are served)")
    _check(fn, heads > 0 and q_heads > 0 and q_heads % heads == 0, f"{q_heads} query heads over {heads} key heads")
    _check(fn, cu.dim() == 1 and cu.shape[0] > 0, "cu is int32 [sequences + 1]")
    cu = _ints(fn, "cu", cu, None)
    n = cu.shape[0] - 1
    _check(fn, cu_k is not None or u == t, f"{t} rows over {u} keys need their offsets cu_k")
    cu_k = cu if cu_k is None else _ints(fn, "cu_k", cu_k, n + 1)
    dev = _same_device(fn, q, k, v, cu, cu_k)
    out = torch.empty((t, q_heads, width), dtype=q.dtype, device=dev)
    if not t or not n:
        return out.zero_()
    _on(dev, lambda st: call(
        "lmoe_prompt_attend", _p(q), q.stride(0), q.stride(1), _p(k), k.stride(0), k.stride(1), _p(v), v.stride(0), v.stride(1),
        dcode(q.dtype), t, u, q_heads, heads, width, _p(cu), _p(cu_k), n, float(width ** -0.5 if scale is None else scale),
        _p(out), st))
    return out
