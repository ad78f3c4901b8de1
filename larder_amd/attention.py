"""Attention of the trunk's rows on MI355X: rotary positions, a paged 8-bit key / value cache, attention of single tokens
over it and of whole prompts. Inference only; every call queues its kernels on the current stream and none waits for the
GPU.

    rotary_freq(width, base, kind, factor, ...)   -> (freq, gain): what rope_rows and append_rows rotate by
    rope_rows(x, positions, freq, ...)            x with each head rotated by its row's position (route_cuda.py:549-591)
    KVCache, KVCache.empty(pages, heads, width)   the cache's four tensors
    append_rows(cache, q, k, v, table, lens, ...) rotates q and k and writes the rows' keys and values into their pages
    read_rows(cache, table, cu, total)            the first tokens of each sequence back in 16 (or 32) bits
    attend_rows(q, cache, table, lens, ...)       the newest rows of each sequence over its cached tokens
    chunk_rows(q, cache, table, lens, cu, ...)    many new rows of each sequence over its cached tokens, causal
    prompt_rows(q, k, v, cu, ...)                 packed sequences, causal, over their own keys and values

Rows are packed: tensors [T, heads, width] hold the sequences one after the other, and cu int32 [sequences + 1] says where
each begins (cu[0] = 0, none less than the one before; one row a sequence where cu is None). Rows of no sequence come back zero.
Heads are 64, 128 or 256 channels wide, and any number of query heads shares a key head. Rows may be strided views, as of a
product that gives q, k and v side by side; one whose layout no kernel reads is copied first. Offsets, lengths and tables live on
the GPU, and the host does not see them: wrong ones give rows and pages of no meaning, and touch no other memory.

lens int32 [sequences] counts a sequence's tokens with the rows of the call among them: row r of n stands at place lens -
n + r. table int32 [sequences, width] lists each sequence's pages in order; entries behind its last page are not read. A
page outside the cache (or the table) holds nothing: no token is written there, attend_rows and chunk_rows see none. read_rows gives its
tokens back as zeros, which prompt_rows would see as any others: a history with such holes is read through a table, and with
offsets, that leave them out (the rows see the keys that are left, as attend_rows has them). Sequences may share pages they
only read; a page that a call writes to stands in one place of one table. A row that sees no token, or only tokens that score
-infinity, attends to nothing: it is zero.
"""
import functools
import math
from typing import NamedTuple

import torch

from . import _lib
from ._lib import call, dcode, stream

__all__ = ["KVCache", "append_rows", "attend_rows", "chunk_rows", "prompt_rows", "read_rows", "rope_rows", "rotary_freq"]


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
        # the ramp may end past the last pair, which is then interpolated in part, as the published one does
        low, high = max(math.floor(pair_of(beta[0])), 0), min(math.ceil(pair_of(beta[1])), width - 1)
        keep = 1.0 - ((torch.arange(width // 2, dtype=torch.float64) - low) / max(high - low, 1e-3)).clamp(0, 1)
        freq = freq * keep + freq / factor * (1.0 - keep)
        gain = 0.1 * math.log(factor) + 1.0
    elif kind not in ("default", "ntk"):
        raise ValueError(f"rotary_freq: {kind!r} is not default, linear, ntk or yarn")
    return freq.to(device), gain


# ---- arguments -------------------------------------------------------------------------------------------------
# A decode step's calls take the host longer than the GPU, so these checks are plain comparisons, and what a refusal says is
# put together only once there is one.

_CODES = (torch.float8_e4m3fn, torch.uint8)
_HALVES = (torch.float16, torch.bfloat16)
_MOST = 2 ** 31 - 1  # of a size that the library takes as an int


def _refuse(fn, why):
    raise ValueError(f"{fn}: {why}")


def _device(fn, first, *others):
    """The index of the one device that every tensor (None: skipped) lives on."""
    dev = first.get_device()
    if dev < 0:
        _refuse(fn, "tensors must live on the GPU")
    for t in others:
        if t is not None and t.get_device() != dev:
            _refuse(fn, "tensors on different devices")
    return dev


_KEYS_APART = 1 << 23  # elements: lmoe_prompt_attend's rows of keys and values are less than that apart


def _rows(fn, name, x, heads=None, width=None, rows=None, apart=1 << 62):
    """(x, row stride, head stride): a [rows, heads, width] tensor the kernels can read (its last axis dense, 16-byte aligned
    rows and heads, rows less than `apart` elements apart), copied if it is not."""
    if x.dim() != 3:
        _refuse(fn, f"{name} is [rows, heads, width], not {tuple(x.shape)}")
    r, h, w = x.shape
    if (heads is not None and h != heads) or (width is not None and w != width) or (rows is not None and r != rows):
        _refuse(fn, f"{name} is [{r}, {h}, {w}]")
    s0, s1, s2 = x.stride()
    s0, s1 = s0 if r > 1 else h * w, s1 if h > 1 else w  # one row's or one head's own stride leads nowhere, and may be anything
    mask = 3 if x.element_size() == 4 else 7
    if s2 != 1 or s0 >= apart or s0 & mask or s1 & mask or x.data_ptr() & 15:
        x = x.contiguous()
        if x.data_ptr() & 15:
            x = x.clone()
        s0, s1 = h * w, w
    return x, s0, s1


def _ints(fn, name, t, n):
    """int32 [n], dense."""
    if t.dtype is not torch.int32 or t.dim() != 1 or t.shape[0] != n:
        _refuse(fn, f"{name} is int32 [{n}], not {t.dtype} {list(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


def _sequences(fn, cu, lens, table, rows):
    """(cu, lens, table, sequences, table width) checked; lens may be None (read_rows)."""
    if table.dtype is not torch.int32 or table.dim() != 2 or table.shape[1] == 0:
        _refuse(fn, f"table is int32 [sequences, pages], not {table.dtype} {list(table.shape)}")
    n, width = table.shape
    if n > _MOST or width > _MOST:
        _refuse(fn, f"{n} sequences of {width} pages are more than an int counts")
    if not table.is_contiguous():
        table = table.contiguous()
    if lens is not None:
        lens = _ints(fn, "lens", lens, n)
    if cu is not None:
        cu = _ints(fn, "cu", cu, n + 1)
    elif rows != n:
        _refuse(fn, f"{rows} rows of {n} sequences need their offsets cu")
    return cu, lens, table, n, width


def _cache(fn, cache):
    k, ks, v, vs = cache
    shape = k.shape
    if len(shape) != 4 or k.dtype not in _CODES or v.dtype is not k.dtype or v.shape != shape:
        _refuse(fn, "the cache's codes are float8_e4m3fn [pages, heads, page, width]")
    if ks.dtype is not torch.float32 or vs.dtype is not torch.float32 or ks.shape != shape[:2] or vs.shape != shape[:2]:
        _refuse(fn, "the cache's scales are float32 [pages, heads]")
    if not (k.is_contiguous() and v.is_contiguous() and ks.is_contiguous() and vs.is_contiguous()):
        _refuse(fn, "the cache's tensors must be contiguous")
    return (*shape, k.data_ptr(), ks.data_ptr(), v.data_ptr(), vs.data_ptr())


def _freq(fn, freq, width):
    if freq is None or freq.dtype is not torch.float64 or freq.dim() != 1 or 2 * freq.shape[0] > width:
        _refuse(fn, "freq is float64 [pairs], two channels a pair")
    return freq if freq.is_contiguous() else freq.contiguous()


def _launch(dev, name, *args):
    """call(name, *args, stream) with dev as the current device."""
    if dev == torch.cuda.current_device():
        return call(name, *args, stream(dev))
    with torch.cuda.device(dev):
        return call(name, *args, stream(dev))


# the workspace of a call is a function of its sizes alone
@functools.lru_cache(maxsize=1024)
def _attend_workspace(*sizes):
    return _lib.lib().lmoe_kv_attend_workspace_bytes(*sizes)


@functools.lru_cache(maxsize=1024)
def _chunk_workspace(*sizes):
    return _lib.lib().lmoe_kv_chunk_workspace_bytes(*sizes)


@functools.lru_cache(maxsize=1024)
def _prompt_workspace(*sizes):
    return _lib.lib().lmoe_prompt_attend_workspace_bytes(*sizes)


# ---- the calls -------------------------------------------------------------------------------------------------

def rope_rows(x, positions, freq, interleaved=False, gain=1.0, out=None):
    """x [T, heads, width] (float16, bfloat16 or float32; width up to 1,024) with the first 2 len(freq) channels of every head
    rotated by the angles positions[t] * freq (positions int32 or int64 [T], any; freq float64, radians): pairs (i, i + len(freq)),
    or (2 i, 2 i + 1) where interleaved, multiplied by gain; the other channels as they are. float32 inside, one rounding.
    out: a tensor of x's shape and type, which may be x (and shares no memory with it otherwise); rows of any strides with a
    dense last axis."""
    fn = "rope_rows"
    if x.dim() != 3:
        _refuse(fn, "x is [rows, heads, width]")
    t, heads, width = x.shape
    dt = dcode(x.dtype)
    if positions.dtype not in (torch.int32, torch.int64) or positions.dim() != 1 or positions.shape[0] != t:
        _refuse(fn, "positions is int32 or int64 [rows]")
    freq = _freq(fn, freq, width)
    if out is None:
        out = x.new_empty((t, heads, width))
    elif out.shape != x.shape or out.dtype is not x.dtype or (width > 1 and out.stride(2) != 1):
        _refuse(fn, "out has x's shape and type and a dense last axis")
    dev = _device(fn, x, positions, freq, out)
    if width > 1 and x.stride(2) != 1:
        x = x.contiguous()
    if not positions.is_contiguous():
        positions = positions.contiguous()
    if x.numel():
        _launch(dev, "lmoe_rope_rows", x.data_ptr(), dt, x.stride(0), x.stride(1), positions.data_ptr(),
                positions.dtype is torch.int64, freq.data_ptr(), freq.shape[0], t, heads, width, bool(interleaved), gain,
                out.data_ptr(), out.stride(0), out.stride(1))
    return out


def append_rows(cache, q, k, v, table, lens, cu=None, freq=None, interleaved=False, gain=1.0, keys=False):
    """Writes the rows k, v [T, heads, width] of each sequence into its pages, k rotated by the rows' places as rope_rows does
    (freq None: as it is), and returns (q, k), tensors of their own: q [T, query heads, width] rotated likewise (None for None),
    and with keys=True the rotated k in its own type, as prompt_rows reads it (else None). float16, bfloat16 or float32. len(freq)
    is a multiple of 8 (of 4 where interleaved). The cache's tensors are written in place."""
    fn = "append_rows"
    pages, heads, page, width, *codes = _cache(fn, cache)
    k, k_row, k_head = _rows(fn, "k", k, heads, width)
    t = k.shape[0]
    v, v_row, v_head = _rows(fn, "v", v, heads, width, t)
    dtype = k.dtype
    dt = dcode(dtype)
    if v.dtype is not dtype or (q is not None and q.dtype is not dtype):
        _refuse(fn, "q, k and v have one type")
    cu, lens, table, n, room = _sequences(fn, cu, lens, table, t)
    pairs = 0
    if freq is not None:
        freq = _freq(fn, freq, width)
        pairs = freq.shape[0]
    dev = _device(fn, k, v, q, table, lens, cu, freq, *cache)
    q_in = q_out = k_out = None
    q_heads = q_row = q_head = 0
    if q is not None:
        q, q_row, q_head = _rows(fn, "q", q, None, width, t)
        q_heads, q_in = q.shape[1], q.data_ptr()
        q_out = q.new_empty((t, q_heads, width))
    if keys:
        k_out = k.new_empty((t, heads, width))
    if t and n:
        _launch(dev, "lmoe_kv_append", q_in, q_row, q_head, q_heads, k.data_ptr(), k_row, k_head, v.data_ptr(), v_row, v_head, dt,
                t, heads, width, None if cu is None else cu.data_ptr(), lens.data_ptr(), n, table.data_ptr(), room, *codes, pages,
                page, None if freq is None else freq.data_ptr(), pairs, bool(interleaved), gain,
                None if q_in is None else q_out.data_ptr(), None if k_out is None else k_out.data_ptr())
    elif t:
        q_out = q_out if q is None else q_out.zero_()
        k_out = k_out if k_out is None else k_out.zero_()
    return q_out, k_out


def read_rows(cache, table, cu, total, dtype=torch.bfloat16):
    """(k, v) [total, heads, width] in dtype: the first cu[b + 1] - cu[b] tokens of every sequence, codes times scale, rounded
    once (bfloat16 holds them exactly): the history that the rows of a later prompt chunk see, for prompt_rows. Tokens whose page
    is not there are zero."""
    fn = "read_rows"
    pages, heads, page, width, *codes = _cache(fn, cache)
    dt = dcode(dtype)
    if cu is None:
        _refuse(fn, "no offsets cu")
    cu, _, table, n, room = _sequences(fn, cu, None, table, total)
    dev = _device(fn, *cache, table, cu)
    k, v = (torch.empty((total, heads, width), dtype=dtype, device=table.device) for _ in range(2))
    if total:
        _launch(dev, "lmoe_kv_read", *codes, pages, page, heads, width, table.data_ptr(), room, cu.data_ptr(), n, total,
                k.data_ptr(), v.data_ptr(), dt)
    return k, v


def attend_rows(q, cache, table, lens, cu=None, most_rows=None, longest=None, scale=None):
    """softmax(scale q k^T) v of the newest rows q [T, query heads, width] (float16 or bfloat16) over the cached tokens of
    their sequences: row r of a sequence's n sees its first lens - n + r + 1 tokens (a row that sees none is zero); scale is
    width^-0.5 if None. Made for few rows a sequence: one token of each, or a speculative decoder's draft.

    Sums are float32; weights are rounded to float16, times 2^11, so that one keeps all its bits down to 2^-25 of the row's
    largest (below about 2^-35 it is zero), and the sum that a row is divided by is the rounded weights'. Values from about 2^90
    on can overflow the sums.

    most_rows and longest size the launch: about the most rows of a sequence (1 without cu, else T / sequences) and tokens of
    one (the table's room). Any values give the same sums in another order."""
    fn = "attend_rows"
    pages, heads, page, width, *codes = _cache(fn, cache)
    q, q_row, q_head = _rows(fn, "q", q, None, width)
    t, q_heads, _ = q.shape
    dtype = q.dtype
    if dtype not in _HALVES:
        _refuse(fn, f"q is float16 or bfloat16, not {dtype}")
    if q_heads == 0 or heads == 0 or q_heads % heads:
        _refuse(fn, f"{q_heads} query heads over {heads} key heads")
    cu, lens, table, n, room = _sequences(fn, cu, lens, table, t)
    dev = _device(fn, q, table, lens, cu, *cache)
    out = q.new_empty((t, q_heads, width))
    if not t or not n:
        return out.zero_()
    most = max(1, min(int(most_rows), t)) if most_rows is not None else 1 if cu is None else -(-t // n)
    long = room * page if longest is None else max(1, min(int(longest), room * page))
    need = _attend_workspace(t, q_heads, heads, width, n, most, long)
    ws = q.new_empty(need, dtype=torch.uint8) if need else None
    _launch(dev, "lmoe_kv_attend", q.data_ptr(), dcode(dtype), q_row, q_head, t, q_heads, heads, width,
            None if cu is None else cu.data_ptr(), lens.data_ptr(), n, table.data_ptr(), room, *codes, pages, page, most, long,
            width ** -0.5 if scale is None else scale, None if ws is None else ws.data_ptr(), need, out.data_ptr())
    return out


def chunk_rows(q, cache, table, lens, cu=None, longest=None, scale=None):
    """softmax(scale q k^T) v of chunks of new rows q [T, query heads, width] (float16 or bfloat16) over the cached tokens of
    their sequences, causal: row r of a sequence's n sees its first lens - n + r + 1 tokens (a row that sees none is zero), as
    attend_rows has it, made for many rows a sequence: a later chunk of a prompt, a message after a long history, a tree of
    drafts. The pages are read as they lie, the chunk's own keys and values among them in the cache's 8 bits. scale is width^-0.5
    if None.

    Sums are float32; weights are rounded to q's type for their product with the values, and the sum that a row is divided by
    is the rounded weights', as in prompt_rows. Keys and values keep all their bits (float16: as long as the scales of two 32-token
    pages beside each other are at most 2^22 apart). Scales of values are powers of two, as append_rows writes them: of others only
    the exponent counts here. A value that is NaN makes its channel NaN in the rows that see it, and touches no other.

    longest sizes the launch: about the most tokens of a sequence (the table's room). Any value gives the same sums in another
    order."""
    fn = "chunk_rows"
    pages, heads, page, width, *codes = _cache(fn, cache)
    q, q_row, q_head = _rows(fn, "q", q, None, width)
    t, q_heads, _ = q.shape
    dtype = q.dtype
    if dtype not in _HALVES:
        _refuse(fn, f"q is float16 or bfloat16, not {dtype}")
    if q_heads == 0 or heads == 0 or q_heads % heads:
        _refuse(fn, f"{q_heads} query heads over {heads} key heads")
    cu, lens, table, n, room = _sequences(fn, cu, lens, table, t)
    dev = _device(fn, q, table, lens, cu, *cache)
    out = q.new_empty((t, q_heads, width))
    if not t or not n:
        return out.zero_()
    long = room * page if longest is None else max(1, min(int(longest), room * page))
    need = _chunk_workspace(t, q_heads, heads, width, n, long)
    ws = q.new_empty(need, dtype=torch.uint8) if need else None
    _launch(dev, "lmoe_kv_chunk", q.data_ptr(), dcode(dtype), q_row, q_head, t, q_heads, heads, width,
            None if cu is None else cu.data_ptr(), lens.data_ptr(), n, table.data_ptr(), room, *codes, pages, page, long,
            width ** -0.5 if scale is None else scale, None if ws is None else ws.data_ptr(), need, out.data_ptr())
    return out


def prompt_rows(q, k, v, cu, cu_k=None, scale=None):
    """softmax(scale q k^T) v of packed sequences, causal: q [T, query heads, width], k and v [U, heads, width] (float16 or
    bfloat16), sequence b's rows cu[b] .. cu[b + 1] of q and cu_k[b] .. cu_k[b + 1] of k and v (cu_k None: the same rows).
    The last row sees all of its sequence's keys, each row before it one fewer; a row that sees none is zero. scale is
    width^-0.5 if None.

    Sums are float32; weights are rounded to the inputs' type for their product with the values (bfloat16: half a step of 2^-8
    each, about as much again as the result's own rounding; float16: times 2^11, as in attend_rows), and the sum that a row is
    divided by is the rounded weights'. A value that is not finite makes its channel infinite or NaN in the rows that see it,
    and touches no other. Values from about 2^100 on can overflow the sums."""
    fn = "prompt_rows"
    q, q_row, q_head = _rows(fn, "q", q)
    t, q_heads, width = q.shape
    k, k_row, k_head = _rows(fn, "k", k, None, width, apart=_KEYS_APART)
    u, heads, _ = k.shape
    v, v_row, v_head = _rows(fn, "v", v, heads, width, u, _KEYS_APART)
    dtype = q.dtype
    if dtype not in _HALVES or k.dtype is not dtype or v.dtype is not dtype:
        _refuse(fn, "q, k and v are all float16 or all bfloat16")
    if width not in (64, 128, 256):
        _refuse(fn, f"heads of {width} channels (64, 128 and 256 are served)")
    if heads == 0 or q_heads == 0 or q_heads % heads:
        _refuse(fn, f"{q_heads} query heads over {heads} key heads")
    n = cu.shape[0] - 1 if cu.dim() == 1 else -1
    if n < 0:
        _refuse(fn, "cu is int32 [sequences + 1]")
    cu = _ints(fn, "cu", cu, n + 1)
    if cu_k is not None:
        cu_k = _ints(fn, "cu_k", cu_k, n + 1)
    elif u != t:
        _refuse(fn, f"{t} rows over {u} keys need their offsets cu_k")
    dev = _device(fn, q, k, v, cu, cu_k)
    out = q.new_empty((t, q_heads, width))
    if not t or not n:
        return out.zero_()
    need = _prompt_workspace(t, u, q_heads, heads, width, n)
    ws = q.new_empty(need, dtype=torch.uint8) if need else None
    _launch(dev, "lmoe_prompt_attend", q.data_ptr(), q_row, q_head, k.data_ptr(), k_row, k_head, v.data_ptr(), v_row, v_head,
            dcode(dtype), t, u, q_heads, heads, width, cu.data_ptr(), (cu if cu_k is None else cu_k).data_ptr(), n,
            width ** -0.5 if scale is None else scale, None if ws is None else ws.data_ptr(), need, out.data_ptr())
    return out
