"""The steps beside the routed experts on T rows: the trunk's 4-bit affine matmul and the shared expert built on it.

    qmv_fits(x, w, scales, group_size, bits, mode, biases)   route_cuda.py:516-522
    qmv_rows(x, w, scales, biases, group_size)               route_cuda.py:525-541 (lmoe_qmv_rows)
    shared_expert_rows(x, gate, up, down)                    mlx_lm's shared_expert MLP on qmv_rows projections
    attention_rows(x, qkv, out, cache, table, lens, ...)     rotary attention on qmv_rows projections and the paged cache

qmv_rows gives every row of x the bits of the reference's kernel (MLX 0.32.4's one-row qmv arithmetic: bf16
weights, bf16 fused multiply-add slots, a float32 slot sum and lane butterfly), reading the weights once a pass.
Weights are MLX's affine 4-bit layout as torch tensors on the GPU: w uint32 / int32 [N, K / 8], scales and biases
bfloat16 [N, K / G].
"""
import torch

from . import attention
from ._lib import call, ptr, stream

__all__ = ["attention_rows", "qmv_fits", "qmv_rows", "shared_expert_rows"]


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
                   most_rows=None, longest=None):
    """The trunk's attention of x [T, H] bf16 (larder_amd.attention's packed rows): out(attend(rotate(qkv(x)))), with qkv and
    out (w, scales, biases, group_size) 4-bit affine weights run through qmv_rows, qkv's output the query heads, then the key
    heads, then the value heads of the cache's width. Nothing else stands between the steps: a model with biases on q, k and v,
    norms of q's and k's heads before the rotation, or a gate on the output calls larder_amd.attention's parts itself. The rows'
    keys and values are written to the cache, then read by

      prompt None              the newest rows of each sequence over its cached tokens (attend_rows; most_rows, longest its)
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
    whole = prompt is True
    cu_k = total = None
    if prompt is not None and not whole:
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
    q, k = attention.append_rows(cache, q, k, v, table, lens, cu=cu, freq=freq, interleaved=interleaved, gain=gain, keys=whole)
    if prompt is None:
        o = attention.attend_rows(q, cache, table, lens, cu=cu, most_rows=most_rows, longest=longest)
    elif whole:
        o = attention.prompt_rows(q, k, v, cu)
    else:
        o = attention.prompt_rows(q, *attention.read_rows(cache, table, cu_k, total, dtype=x.dtype), cu, cu_k=cu_k)
    return qmv_rows(o.reshape(t, q_heads * width), *out)
