"""The public entry points, with the reference's names and signatures
(src/fold_attention/interface.py:106-173).

Training: `fold_attn_func` and `fold_attn_varlen_func` run the library's
forward and its deterministic backward, whose gradients are the same bits
however the GPU schedules them and whatever a request is batched with.

Serving: `fold_attn_with_kvcache` attends over a `FoldKVCache`, optionally
appending one token per request first.
"""

from __future__ import annotations

import math

import torch

from .backward.launch import attention_forward, prepare_backward, window_backward, window_forward
from .utils import check_status as read_status
from .utils import check_window, require_sm100

# Set to True to read the backward's device status word after every backward (one host
# synchronisation each) and raise FoldLibraryError if a kernel gave up a bounded wait; by
# default nothing in the training path synchronises, as in the reference.
check_status = False


def _check_qkv(q, k, v, ndim):
    if q.ndim != ndim or k.ndim != ndim or v.ndim != ndim:
        raise ValueError(f"q, k and v must have {ndim} dimensions")
    if q.shape[0] != k.shape[0] or k.shape != v.shape:
        raise ValueError("q, k and v must have compatible shapes")
    if q.shape[-1] != k.shape[-1] or q.shape[-2] % k.shape[-2]:
        raise ValueError(
            "head dims must match and the query heads must be a multiple of the KV heads"
        )
    if q.dtype not in (torch.bfloat16, torch.float16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("q, k and v must share a bf16 or fp16 dtype")
    if q.device != k.device or q.device != v.device or q.device.type != "cuda":
        raise ValueError("q, k and v must be on the same CUDA device")
    require_sm100(q.device)


def _windowed_input(x):
    """`x` as the windowed kernels read it in place, or a copy: a contiguous head
    dim, rows on 16-byte boundaries, and no axis that a broadcast gave stride 0."""
    st = x.stride()
    ok = st[-1] == 1 and all(s and s % 8 == 0 for s in st[:-1]) and x.data_ptr() % 16 == 0
    return x if ok else x.clone(memory_format=torch.contiguous_format)


class _FoldAttnFunc(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, softmax_scale, causal, window, sinks):
        if window:
            q, k, v = _windowed_input(q), _windowed_input(k), _windowed_input(v)
            out, lse, rest = window_forward(q, k, v, window, sinks, softmax_scale, grad=any(ctx.needs_input_grad))
        else:
            rest = None
            q, k, v = (x if x.stride(-1) == 1 else x.contiguous() for x in (q, k, v))
            out, lse = attention_forward(q, k, v, causal=causal, softmax_scale=softmax_scale)
        ctx.save_for_backward(q, k, v, out, lse, rest)
        ctx.softmax_scale, ctx.causal, ctx.window, ctx.sinks = softmax_scale, causal, window, sinks
        return out

    @staticmethod
    def backward(ctx, *grad_outputs):
        (dout,) = grad_outputs
        q, k, v, out, lse, rest = ctx.saved_tensors
        if ctx.window:
            dq, dk, dv, status = window_backward(q, k, v, out, rest, _windowed_input(dout), lse, ctx.window, ctx.sinks, ctx.softmax_scale)
            if check_status:
                read_status(status.view(torch.int32), "fold_attn_func's backward")
            return dq, dk, dv, None, None, None, None
        run = prepare_backward(
            q.transpose(1, 2),
            k.transpose(1, 2),
            v.transpose(1, 2),
            out.transpose(1, 2),
            dout.contiguous().transpose(1, 2),
            lse,
            causal=ctx.causal,
            softmax_scale=ctx.softmax_scale,
        )
        dq, dk, dv = run()
        if check_status:
            run.check()
        return dq.transpose(1, 2), dk.transpose(1, 2), dv.transpose(1, 2), None, None, None, None


class _FoldAttnVarlenFunc(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu_seqlens, max_seqlen, softmax_scale, causal, window, sinks):
        if window:
            q, k, v = _windowed_input(q), _windowed_input(k), _windowed_input(v)
            out, lse, rest = window_forward(
                q, k, v, window, sinks, softmax_scale, cu_seqlens, max_seqlen, grad=any(ctx.needs_input_grad))
        else:
            rest = None
            q, k, v = (x if x.stride(-1) == 1 else x.contiguous() for x in (q, k, v))
            out, lse = attention_forward(
                q, k, v, causal=causal, softmax_scale=softmax_scale,
                cu_seqlens=cu_seqlens, max_seqlen=max_seqlen,
            )
        ctx.save_for_backward(q, k, v, out, lse, cu_seqlens, rest)
        ctx.max_seqlen, ctx.softmax_scale, ctx.causal = max_seqlen, softmax_scale, causal
        ctx.window, ctx.sinks = window, sinks
        return out

    @staticmethod
    def backward(ctx, *grad_outputs):
        (dout,) = grad_outputs
        q, k, v, out, lse, cu_seqlens, rest = ctx.saved_tensors
        if ctx.window:
            dq, dk, dv, status = window_backward(
                q, k, v, out, rest, _windowed_input(dout), lse, ctx.window, ctx.sinks, ctx.softmax_scale, cu_seqlens, ctx.max_seqlen)
            if check_status:
                read_status(status.view(torch.int32), "fold_attn_varlen_func's backward")
            return dq, dk, dv, None, None, None, None, None, None
        run = prepare_backward(
            q,
            k,
            v,
            out,
            dout.contiguous(),
            lse,
            causal=ctx.causal,
            softmax_scale=ctx.softmax_scale,
            cu_seqlens=cu_seqlens,
            max_seqlen=ctx.max_seqlen,
        )
        dq, dk, dv = run()
        if check_status:
            run.check()
        return dq, dk, dv, None, None, None, None, None, None


def fold_attn_func(q, k, v, softmax_scale=None, causal=False, window=None, sinks=0):
    """Self-attention over `(batch, seqlen, nheads, headdim)` tensors.

    `k` and `v` may have fewer heads than `q` (GQA/MQA). Returns the output,
    shaped and typed as `q`. The backward reduces across CTAs in integers, so
    the gradients do not depend on the order work runs in. Head dims 64, 96
    and 128, bf16 or fp16, SM100.

    `window` (with `causal=True`) is a sliding window: the query at position i
    sees the `window` newest keys up to its own, `i - window < j <= i`, and the
    sequence's first `sinks` keys. The work is the window's, not the
    sequence's, and the gradients keep their order-free bits. Where every
    query sees one key, dq and dk are zero.
    """
    window, sinks = check_window(window, sinks, causal)
    _check_qkv(q, k, v, 4)
    if q.shape[1] != k.shape[1]:
        raise ValueError("self-attention needs equal query and key lengths")
    scale = 1.0 / math.sqrt(q.shape[-1]) if softmax_scale is None else float(softmax_scale)
    return _FoldAttnFunc.apply(q, k, v, scale, bool(causal), window, sinks)


def fold_attn_varlen_func(
    q,
    k,
    v,
    cu_seqlens_q,
    cu_seqlens_k=None,
    max_seqlen_q=None,
    max_seqlen_k=None,
    softmax_scale=None,
    causal=False,
    window=None,
    sinks=0,
):
    """Self-attention over sequences packed along the first axis.

    `q` is `(total, nheads, headdim)` and `k`, `v` `(total, nheads_k,
    headdim)`, split by `cu_seqlens_q`, a CUDA int32 `(batch + 1,)` tensor.
    The keys are the queries' own sequences, so `cu_seqlens_k` and
    `max_seqlen_k` may be left out; if given they must match. A request's
    gradients are the same bits alone and packed with others. `window` and
    `sinks` as for `fold_attn_func`, counted within each sequence; with a window,
    rows behind the last sequence give zeros, and have zeros for gradients.
    """
    window, sinks = check_window(window, sinks, causal)
    _check_qkv(q, k, v, 3)
    cu = cu_seqlens_q
    if cu.ndim != 1 or cu.dtype != torch.int32 or cu.device != q.device:
        raise ValueError("cu_seqlens_q must be a CUDA int32 vector on q's device")
    if cu_seqlens_k is not None and cu_seqlens_k is not cu and not torch.equal(cu_seqlens_k, cu):
        raise ValueError("self-attention needs cu_seqlens_k == cu_seqlens_q")
    if max_seqlen_q is None:
        max_seqlen_q = int(torch.diff(cu).max())
    if max_seqlen_k is not None and int(max_seqlen_k) != int(max_seqlen_q):
        raise ValueError("self-attention needs max_seqlen_k == max_seqlen_q")
    scale = 1.0 / math.sqrt(q.shape[-1]) if softmax_scale is None else float(softmax_scale)
    return _FoldAttnVarlenFunc.apply(q, k, v, cu.contiguous(), int(max_seqlen_q), scale, bool(causal), window, sinks)


def fold_attn_with_kvcache(q, cache, k=None, v=None, cu_seqlens=None, lens=None):
    """Attention of one query token per request over `cache`, or of a chunk of
    new tokens per request.

    `q` is `(batch, nheads, headdim)` or `(batch, 1, nheads, headdim)`. With
    `k` and `v` (`(batch, nheads_k, headdim)`, or with the extra axis of 1)
    the token is appended first, so the query sees it. Returns the output in
    `q`'s shape and dtype.

    With `cu_seqlens` (int32 `(batch + 1,)` on the device; `lens` the host's copy
    of the counts, without which the call waits for the device) `q` is `(total,
    nheads, headdim)`, each request's new tokens packed, and `k` and `v` `(total,
    nheads_k, headdim)`: they are appended, and each query sees the keys up to its
    own (`FoldKVCache.extend`). Without `k` and `v` the cache already holds them.
    """
    if (k is None) != (v is None):
        raise ValueError("k and v are both given or both left out")
    if cu_seqlens is not None:
        return cache.attend_chunk(q, cu_seqlens, lens) if k is None else cache.extend(q, k, v, cu_seqlens, lens)
    if lens is not None:
        raise ValueError("lens are the counts that cu_seqlens describes: give both")
    squeeze = q.ndim == 4
    if squeeze and q.shape[1] != 1:
        raise ValueError("fold_attn_with_kvcache takes one query token per request")
    if squeeze:
        q = q[:, 0]
    if k is None:
        out = cache.attend(q)
    else:
        out = cache.decode(q, k[:, 0] if squeeze else k, v[:, 0] if squeeze else v)
    return out[:, None] if squeeze else out
