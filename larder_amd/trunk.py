"""The steps beside the routed experts on T rows: the trunk's 4-bit affine matmul and the shared expert built on it.

    qmv_fits(x, w, scales, group_size, bits, mode, biases)   route_cuda.py:516-522
    qmv_rows(x, w, scales, biases, group_size)               route_cuda.py:525-541 (lmoe_qmv_rows)
    shared_expert_rows(x, gate, up, down)                    mlx_lm's shared_expert MLP on qmv_rows projections
    attention_rows(x, qkv, out, cache, table, lens, ...)     rotary attention on qmv_rows projections and the paged cache,
                                                             its heads normed first where asked
    norm_rows(x, weight, eps, residual, group, total)        root-mean-square norm, after the residual's addition
    read_codes(codes, scales, dtype)                         rows that norm_rows gave in 8 bits

qmv_rows gives every row of x the bits of the reference's kernel (MLX 0.32.4's one-row qmv arithmetic: bf16
weights, bf16 fused multiply-add slots, a float32 slot sum and lane butterfly), reading the weights once a pass.
Weights are MLX's affine 4-bit layout as torch tensors on the GPU: w uint32 / int32 [N, K / 8], scales and biases
bfloat16 [N, K / G].
"""
import torch

from . import attention
from ._lib import F32, call, dcode, ptr, stream

__all__ = ["attention_rows", "norm_rows", "qmv_fits", "qmv_rows", "read_codes", "shared_expert_rows"]


def qmv_fits(x, w, scales, group_size, bits, mode, biases):
    """Whether qmv_rows serves this product (route_cuda.py:516-522): 4-bit affine with biases, bf16 x, scales and
    biases, a 2-D packed weight, K a multiple of 16 and of the group size, the group size a multiple of 16."""
    k = x.shape[-1]
    return (bits == 4 and mode == "affine" and biases is not None and x.dtype == torch.bfloat16
            and scales.dtype == torch.bfloat16 and biases.dtype == torch.bfloat16
            and w.dtype in (torch.int32, torch.uint32) and w.dim() == 2 and k % 16 == 0 and k % group_size == 0
            and group_size % 16 == 0 and w.shape[-1] * 8 == k)


def qmv_rows(x, w, scales, biases, group_size):
    """x [..., T, K] bf16 times the 4-bit affine weight (transposed) -> [..., T, N] bf16, each row bit-equal to the
    reference's one-row pass (route_cuda.py:525-541)."""
    if not qmv_fits(x, w, scales, group_size, 4, "affine", biases):
        raise ValueError("qmv_rows: bf16 x, 4-bit affine uint32 weights with bf16 scales and biases, K a multiple of "
                         "16 and of the group size")
    K = x.shape[-1]
    N = w.shape[0]
    x2 = x.reshape(-1, K).contiguous()
    out = torch.empty((x2.shape[0], N), dtype=torch.bfloat16, device=x.device)
    w, scales, biases = w.contiguous(), scales.contiguous(), biases.contiguous()  # copies live until the launch is out
    call("lmoe_qmv_rows", ptr(x2), x2.shape[0], ptr(w), ptr(scales), ptr(biases), N, K, group_size, ptr(out), stream())
    return out.reshape(x.shape[:-1] + (N,))


def shared_expert_rows(x, gate, up, down):
    """mlx_lm's shared-expert MLP, down(silu(gate(x)) * up(x)), for x [..., T, H] bf16 with each projection a
    (w, scales, biases, group_size) 4-bit affine weight run through qmv_rows; the SwiGLU rounds once to bf16
    (lmoe_swiglu_bf16). The sigmoid-gated add to the routed output is route.tail's."""
    (wg, sg, bg, gs), (wu, su, bu, us) = gate, up
    if gs == us and wg.shape == wu.shape and qmv_fits(x, wg, sg, gs, 4, "affine", bg) and qmv_fits(
            x, wu, su, us, 4, "affine", bu):  # gate, up and the SwiGLU in one launch
        K, N = x.shape[-1], wg.shape[0]
        x2 = x.reshape(-1, K).contiguous()
        h = torch.empty((x2.shape[0], N), dtype=torch.bfloat16, device=x.device)
        held = [t.contiguous() for t in (wg, sg, bg, wu, su, bu)]  # strided ones' copies, alive until the launch is out
        call("lmoe_qmv_swiglu_rows", ptr(x2), x2.shape[0], *map(ptr, held), N, K, gs, ptr(h), stream())
        return qmv_rows(h.reshape(x.shape[:-1] + (N,)), *down)
    g = qmv_rows(x, *gate)
    u = qmv_rows(x, *up)
    h = torch.empty_like(g)
    call("lmoe_swiglu_bf16", ptr(g), ptr(u), g.numel(), ptr(h), stream())
    return qmv_rows(h, *down)


def attention_rows(x, qkv, out, cache, table, lens, cu=None, freq=None, interleaved=False, gain=1.0, prompt=None,
                   most_rows=None, longest=None, norms=None):
    """The trunk's attention of x [T, H] bf16 (larder_amd.attention's packed rows): out(attend(rotate(norm(qkv(x))))), with qkv and
    out (w, scales, biases, group_size) 4-bit affine weights run through qmv_rows, qkv's output the query heads, then the key
    heads, then the value heads of the cache's width. norms (query weight, key weight, eps): the heads of q and k are normed by
    norm_rows before their rotation (None: they are not). Nothing else stands between the steps: a model with biases on q, k and
    v, or a gate on the output calls larder_amd.attention's parts itself. The rows' keys and values are written to the cache,
    then read by

      prompt None              the newest rows of each sequence over its cached tokens (attend_rows; most_rows, longest its)
      prompt "chunk"           many new rows of each sequence over its cached tokens, straight from the pages: a prompt's first
                               or a later chunk (chunk_rows; longest its). All keys and values are in the cache's 8 bits
      prompt True              sequences that begin with this call, over the call's own keys and values (prompt_rows)
      prompt (cu_k, total)     later chunks of prompts: over all the cached tokens, lens of each, total in all, cu_k int32
                               [sequences + 1] where each begins (read_rows, prompt_rows); none of them in a page that is
                               not there. The chunk's own keys and values are among them, in the cache's 8 bits, where a
                               first chunk (True) takes its own in 16
    """
    heads, width = cache.k.shape[1], cache.k.shape[3]
    # what a later call would refuse is refused here, before the cache is written
    if prompt is not None and cu is None:
        raise ValueError("attention_rows: a prompt's rows need their offsets cu")
    whole, chunk = prompt is True, prompt == "chunk" if isinstance(prompt, str) else False
    if isinstance(prompt, str) and not chunk:
        raise ValueError(f"attention_rows: prompt {prompt!r} is not \"chunk\"")
    cu_k = total = None
    if prompt is not None and not whole and not chunk:
        cu_k, total = prompt
        cu_k = attention._ints("attention_rows", "cu_k", cu_k, table.shape[0] + 1)
        if cu_k.device != x.device or total < 0:
            raise ValueError("attention_rows: cu_k lives where x does, and total is no less than zero")
    y = qmv_rows(x, *qkv)
    t, q_heads = y.shape[0], y.shape[1] // width - 2 * heads
    if q_heads <= 0 or y.shape[1] % width or heads == 0 or q_heads % heads:
        raise ValueError(f"attention_rows: {y.shape[1]} outputs are not query heads and {heads} key and value heads of {width}")
    w, scales, biases, group_size = out
    if not qmv_fits(y[:, :q_heads * width], w, scales, group_size, 4, "affine", biases):
        raise ValueError(f"attention_rows: out is a 4-bit affine weight of {q_heads} heads of {width}")
    q, k, v = y.view(t, y.shape[1] // width, width).split([q_heads, heads, heads], 1)
    if norms is not None:
        q, k = norm_rows(q, norms[0], norms[2]), norm_rows(k, norms[1], norms[2])
    q, k = attention.append_rows(cache, q, k, v, table, lens, cu=cu, freq=freq, interleaved=interleaved, gain=gain, keys=whole)
    if prompt is None:
        o = attention.attend_rows(q, cache, table, lens, cu=cu, most_rows=most_rows, longest=longest)
    elif chunk:
        o = attention.chunk_rows(q, cache, table, lens, cu, longest=longest)
    elif whole:
        o = attention.prompt_rows(q, k, v, cu)
    else:
        o = attention.prompt_rows(q, *attention.read_rows(cache, table, cu_k, total, dtype=x.dtype), cu, cu_k=cu_k)
    return qmv_rows(o.reshape(t, q_heads * width), *out)


def _planes(x):
    """(x, rows, heads, row stride, head stride): x [..., H] as rows of heads, its last axis dense; copied where its leading
    axes are not two strides."""
    n, st = x.dim(), x.stride()
    if n > 3 or (st[-1] != 1 and x.shape[-1] > 1):
        x = x.contiguous()
        st = x.stride()
    if n == 2:
        return x, x.shape[0], 1, st[0], 0
    if n == 3:
        return x, x.shape[0], x.shape[1], st[0], st[1]
    return x, x.numel() // x.shape[-1], 1, x.shape[-1], 0


def norm_rows(x, weight, eps=1e-6, residual=None, group=None, total=None):
    """Root-mean-square norm over the last axis of x [..., H] (float16, bfloat16 or float32; the residual stream, or the heads of
    q and k before their rotation): with s = x + residual, y = s / sqrt(mean(s^2) + eps) * weight. weight [H] in x's type or
    float32, residual of x's shape and type. Views with a dense last axis are read as they lie. float32 inside: y is of the sum
    before that is rounded, and rows whose squares pass float32 (from about 2^64 / sqrt(H) on) keep their values.

    group None: y in x's type. Else y in 8 bits, as (codes float8_e4m3fn, scales float32 [..., H / group]): the scale of `group`
    neighbouring channels (32, 64, 128, 256 or 512 that divide H, or H itself) is the least power of two (2^-100 or more) that
    brings their largest finite magnitude to 448 or less, and infinities and NaN are kept as NaN. read_codes gives the rows back.
    With a residual (or total) the result is followed by s in x's type, rounded once, in total, if that is given: a tensor
    of x's shape and type with a dense last axis, which may be x or the residual (and shares no memory with them otherwise)."""
    fn = "norm_rows"
    if x.dim() == 0 or x.shape[-1] == 0:
        attention._refuse(fn, "x is [..., channels]")
    shape, dtype = x.shape, x.dtype
    h, plain = shape[-1], len(shape) == 2  # [rows, channels]: the most common, with the host's time in mind
    dt = dcode(dtype)
    if weight.dim() != 1 or weight.shape[0] != h or (weight.dtype is not dtype and weight.dtype is not torch.float32):
        attention._refuse(fn, f"weight is [{h}] in x's type or float32, not {weight.dtype} {list(weight.shape)}")
    if not 0.0 < eps < float("inf"):
        attention._refuse(fn, f"eps {eps} is not above zero")
    if residual is not None and (residual.shape != shape or residual.dtype is not dtype):
        attention._refuse(fn, "residual has x's shape and type")
    if group is not None and group != h and (group not in (32, 64, 128, 256, 512) or h % group):
        attention._refuse(fn, f"scales of {group} channels in rows of {h} (32, 64, 128, 256 or 512 that divide them, or whole rows)")
    sums = residual is not None or total is not None
    own = total is None  # the sum's tensor is this call's
    if own:
        total = x.new_empty(shape) if sums else None
    elif total.shape != shape or total.dtype is not dtype or (h > 1 and total.stride(-1) != 1) or (
            total.dim() > 3 and not total.is_contiguous()):
        attention._refuse(fn, "total has x's shape and type and a dense last axis")
    elif any(s == 0 and n > 1 for s, n in zip(total.stride(), shape)):
        attention._refuse(fn, "total has a place for every element")
    dev = attention._device(fn, x, weight, residual, total)
    if h > 1 and weight.stride(0) != 1:
        weight = weight.contiguous()
    x, t, heads, x_row, x_head = _planes(x)
    r_row = r_head = s_row = s_head = 0
    if h > attention._MOST or heads > attention._MOST:
        attention._refuse(fn, f"{heads} heads of {h} channels are more than an int counts")
    if residual is not None:
        residual, _, _, r_row, r_head = _planes(residual)
    if total is not None:
        s_row, s_head = (h, 0) if own and plain else _planes(total)[3:]
    scales = None
    if group is None:
        out = x.new_empty(shape)
    else:
        out = x.new_empty(shape, dtype=torch.float8_e4m3fn)
        scales = x.new_empty(shape[:-1] + (h // group,), dtype=torch.float32)
    if t and heads:
        attention._launch(dev, "lmoe_norm_rows", x.data_ptr(), dt, x_row, x_head, None if residual is None else residual.data_ptr(),
                          r_row, r_head, weight.data_ptr(), dt if weight.dtype is dtype else F32, t, heads, h, eps, out.data_ptr(),
                          0 if group is None else group, None if scales is None else scales.data_ptr(),
                          None if total is None else total.data_ptr(), s_row, s_head)
    if group is None:
        return (out, total) if sums else out
    return (out, scales, total) if sums else (out, scales)


def read_codes(codes, scales, dtype=torch.bfloat16):
    """Rows in dtype from the 8 bits that norm_rows gave: codes float8_e4m3fn [..., H] times scales float32 [..., H / group], each
    rounded once (bfloat16 holds them exactly)."""
    fn = "read_codes"
    if codes.dtype not in attention._CODES or codes.dim() == 0 or codes.shape[-1] == 0:
        attention._refuse(fn, "codes are float8_e4m3fn [..., channels]")
    if scales.dtype is not torch.float32 or scales.dim() != codes.dim() or scales.shape[:-1] != codes.shape[:-1] or (
            scales.shape[-1] == 0 or codes.shape[-1] % scales.shape[-1]):
        attention._refuse(fn, f"scales are float32 {list(codes.shape[:-1])} and a divisor of {codes.shape[-1]}, not "
                              f"{scales.dtype} {list(scales.shape)}")
    if codes.shape[-1] > attention._MOST:
        attention._refuse(fn, f"rows of {codes.shape[-1]} channels are more than an int counts")
    dt = dcode(dtype)
    dev = attention._device(fn, codes, scales)
    codes, scales = codes.contiguous(), scales.contiguous()
    if codes.data_ptr() & 15:
        codes = codes.clone()
    out = codes.new_empty(codes.shape, dtype=dtype)
    if codes.numel():
        attention._launch(dev, "lmoe_read_codes", codes.data_ptr(), scales.data_ptr(), codes.numel(),
                          codes.shape[-1] // scales.shape[-1], out.data_ptr(), dt)
    return out
