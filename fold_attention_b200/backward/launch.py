"""The backward's host side: bind one call's tensors, return the launch.

Mirrors `prepare_backward` of the reference
(src/fold_attention/backward/launch.py:75-117): the launch returns `(dq, dk,
dv)`, the same tensors on every call, and owns its workspace, so two captured
graphs never share one. All device work goes through the C ABI
(`fold_bwd_run`): preprocess, main loop, postprocess on the current stream,
with no host synchronisation.
"""

from __future__ import annotations

import ctypes
import functools
import math
from dataclasses import dataclass

import torch

from .. import _lib
from ..utils import Launch, check_status, check_window
from .plan import Plan, plan_dense, plan_varlen, tile_config

P, I, F, Z = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_size_t
_lib.register("fold_bwd_workspace_bytes", [I, I, I, I, I, I, I, I, I], Z)
_lib.register("fold_bwd_workspace_layout", [I, I, I, I, I, I, I, I, I, P])
_lib.register(
    "fold_bwd_run",
    [P, P, P, P, P, P, P, P, P, P, P, I, I, I, I, I, I, I, I, F, P, Z, I, I, I, P],
)
_lib.register(
    "fold_bwd_run_phases",
    [P, P, P, P, P, P, P, P, P, P, P, I, I, I, I, I, I, I, I, F, P, Z, I, I, I, I, P],
)
_lib.register(
    "fold_bwd_window",
    [P, P, P, P, P, P, P, P, P, P, P, P, I, I, I, I, I, I, I, F, P, Z, I, I, I, I, P],
)
_lib.register("fold_bwd_window_layout", [I, I, I, I, I, I, I, I, I, P])
_lib.register("fold_bwd_counters", [P, I])
_lib.register("fold_wait_probe", [ctypes.c_longlong, P, P, P])
_lib.register("fold_fwd_run", [P, P, P, P, P, P, P, I, I, I, I, I, I, I, I, F, P])
_lib.register("fold_fwd_window", [P, P, P, P, P, P, P, P, I, I, I, I, I, I, I, F, I, I, P, I, P])
_lib.register("fold_fwd_window_sm100", [P, P, P, P, P, P, P, P, I, I, I, I, I, I, I, F, I, I, P, I, P, P])
_lib.register("fold_fwd_sm100_supported", [I, I])
_lib.register("fold_fwd_run_sm100", [P, P, P, P, P, P, P, I, I, I, I, I, I, I, I, F, P, P])

KERNELS = {"auto": 0, "mma": 1, "sm100": 2}


@dataclass(eq=False)
class BackwardLaunch(Launch):
    """`prepare_backward`'s result: calling it returns `(dq, dk, dv)`."""

    plan: Plan | None = None
    workspace: torch.Tensor | None = None
    layout: tuple | None = None


def _strides(tensors, varlen):
    """(batch, row, head) element strides of `(B, H, S, D)` views or packed
    `(total, H, D)` tensors, as a host int64 array."""
    out = []
    for t in tensors:
        if t.stride(-1) != 1:
            raise ValueError("the head dim must be contiguous")
        if varlen:
            out += [0, t.stride(0), t.stride(1)]
        else:
            out += [t.stride(0), t.stride(2), t.stride(1)]
    return (ctypes.c_int64 * len(out))(*out)


def prepare_backward(
    q,
    k,
    v,
    o,
    do,
    lse,
    *,
    causal,
    softmax_scale=None,
    cu_seqlens=None,
    max_seqlen=None,
    out_dtype=None,
    plan: Plan | None = None,
    kernel: str = "auto",
    window=None,
    sinks=0,
    o_rest=None,
):
    """Bind dQ, dK and dV of causal or full self-attention to one call's
    tensors, and return the launch that computes them.

    Dense: `(B, H, S, D)` views and `lse` `(B, H, S)`. Varlen: `(total, H, D)`
    packed by `cu_seqlens` `(B + 1,)` int32, and `lse` `(H, total)`. `lse` is
    in nats. `kernel` picks the main loop: "auto" (tcgen05 where it applies),
    "mma" or "sm100". `plan` cuts the work (`plan_dense` / `plan_varlen` by
    default): the tcgen05 main loop takes any `Plan`, the mma.sync one only
    whole groups over whole query ranges.

    `window` and `sinks` (causal calls): query i sees key j when `i - j <
    window` or `j < sinks`. A windowed call cuts its own work and takes no
    `plan`: key blocks past the sinks stay private to a CTA, the sinks' blocks
    meet every later query and fold on the integer grids. `o_rest` is
    `attention_forward`'s remainder of O, laid out as `o`: with it Delta is exact where
    queries see few keys (`REST_KEYS` says what that is worth).
    """
    window, sinks = check_window(window, sinks, causal)
    if o_rest is not None and not window:
        raise ValueError("o_rest is a windowed call's: give a window")
    if window and plan is not None:
        raise NotImplementedError("a windowed backward cuts its own work: it takes no plan")
    varlen = cu_seqlens is not None
    if varlen:
        total, H, D = q.shape
        H_KV = k.shape[1]
        B = cu_seqlens.shape[0] - 1
        if max_seqlen is None:
            max_seqlen = int(torch.diff(cu_seqlens).max())
        S = int(max_seqlen)
    else:
        B, H, S, D = q.shape
        H_KV = k.shape[1]
        total = B * S
        if k.shape[2] != S:
            raise NotImplementedError("the integer grids assume self-attention")
    if v.shape[-1] != D:
        raise NotImplementedError("the value head dim must equal the key head dim")
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("q, k and v must be bf16 or fp16")
    # the kernels index every tensor by q's sizes: anything that does not match would be read or written past its end
    lead = (total,) if varlen else (B,)
    if k.dim() != q.dim() or tuple(k.shape[:1]) != lead or k.shape[-1] != D or v.shape != k.shape:
        raise ValueError(f"k and v {tuple(k.shape)}, {tuple(v.shape)} do not match q {tuple(q.shape)}")
    if o.shape != q.shape or do.shape != q.shape:
        raise ValueError(f"o and do are q's shape {tuple(q.shape)} (got {tuple(o.shape)}, {tuple(do.shape)})")
    if o_rest is not None and (o_rest.shape != o.shape or o_rest.stride() != o.stride() or o_rest.dtype != q.dtype or o_rest.device != q.device):
        raise ValueError(f"o_rest is laid out as o, {tuple(o.shape)} by {o.stride()} in {q.dtype} "
                         f"(got {tuple(o_rest.shape)} by {o_rest.stride()} in {o_rest.dtype})")
    if tuple(lse.shape) != ((H, total) if varlen else (B, H, S)):
        raise ValueError(f"lse is {'(H, total)' if varlen else '(B, H, S)'} (got {tuple(lse.shape)})")
    if any(t.dtype != q.dtype for t in (k, v, o, do)):
        raise ValueError("q, k, v, o and do must be the same 16-bit type")
    if any(t.device != q.device for t in (k, v, o, do, lse)) or any(t.stride(-1) != 1 for t in (q, k, v, o, do)):
        raise ValueError("q, k, v, o, do and lse are on one device, each with a contiguous head dim")
    if varlen and (cu_seqlens.dtype != torch.int32 or cu_seqlens.device != q.device):
        raise ValueError("cu_seqlens is int32 on q's device")
    if H % H_KV:
        raise ValueError("the query heads must be a multiple of the KV heads")
    if D not in (64, 96, 128):
        raise NotImplementedError(f"head_dim {D}: 64, 96 and 128 are supported")
    if out_dtype is not None and out_dtype != q.dtype:
        raise NotImplementedError("gradients are returned in the inputs' dtype")
    dev = q.device
    sm = float(softmax_scale) if softmax_scale is not None else 1.0 / math.sqrt(D)
    if kernel not in KERNELS:
        raise ValueError(f"kernel is one of {tuple(KERNELS)}")
    G = H // H_KV
    cfg = tile_config(D, kernel)
    if window:
        plan = Plan(G, 0)
    elif plan is None:
        plan = plan_varlen(H, H_KV, cfg) if varlen else plan_dense(B, H, H_KV, S, D, bool(causal), cfg)
    if plan.subgroup < 1 or G % plan.subgroup or plan.record < 0:
        raise ValueError(f"a plan of {plan.subgroup} heads per work item for groups of {G}")
    if plan.folds(G) and cfg.tile_n != 128:
        raise NotImplementedError(
            "the mma.sync main loop keeps a key block's dK and dV in one CTA: its plan is the whole group over the whole range")
    lse = lse.contiguous()
    if lse.dtype != torch.float32:
        raise ValueError("lse must be fp32")
    dq, dk, dv = (torch.empty_like(x) for x in (q, k, v))
    lay = (ctypes.c_int64 * 12)()
    if window:
        _lib.call("fold_bwd_window_layout", B, H, H_KV, S, total, D, int(varlen), window, sinks, lay)
        nbytes = lay[11]
    else:
        nbytes = _lib.lib.fold_bwd_workspace_bytes(B, H, H_KV, S, total, D, int(varlen), plan.subgroup, plan.record)
        _lib.call("fold_bwd_workspace_layout", B, H, H_KV, S, total, D, int(varlen), plan.subgroup, plan.record, lay)
    workspace = torch.empty(nbytes, device=dev, dtype=torch.uint8)
    tensors = (q, k, v, o, do, dq, dk, dv)
    strides = _strides(tensors, varlen)
    cu = cu_seqlens
    args = (
        q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), do.data_ptr(), lse.data_ptr(),
        dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), ctypes.addressof(strides),
        _lib.ptr(cu), B, H, H_KV, S, total, D, int(bool(causal)),
        int(q.dtype == torch.float16), sm, workspace.data_ptr(), nbytes, KERNELS[kernel],
        plan.subgroup, plan.record,
    )

    if window:   # the same arguments without the mask and the plan, and O as it was rounded
        args = (*args[:4], _lib.ptr(o_rest), *args[4:17], *args[18:23], window, sinks)

    def run():
        if window:
            run_phase(15)
        else:
            _lib.call("fold_bwd_run", *args, _lib.stream(dev))
        return dq, dk, dv

    def run_phase(phases):
        """One or more of the backward's phases (1 preprocess, 8 work list,
        2 main loop, 4 postprocess; in that order), for callers that time them
        apart or look at the work list between them."""
        if window:
            with _lib.on(dev):
                _lib.call("fold_bwd_window", *args, int(phases), _lib.stream(dev))
        else:
            _lib.call("fold_bwd_run_phases", *args, int(phases), _lib.stream(dev))

    held = (q, k, v, o, o_rest, do, lse, dq, dk, dv, workspace, cu, strides)
    launch = BackwardLaunch(run, held, plan, workspace, tuple(lay[:11]))
    launch.run_phase = run_phase
    launch.status = workspace[lay[5]: lay[5] + 4].view(torch.int32)
    # the work list as the device built it (n_items, 8): key block, KV head, request, first head,
    # heads, first / one-past-last query block, cost in tiles; and, for a folding plan, the integer
    # dK and dV accumulators [H_KV, padded rows, D]
    launch.work = workspace[lay[9]: lay[9] + 32 * lay[10]].view(torch.int32).view(-1, 8)
    launch.dk_acc = launch.dv_acc = None
    if lay[8]:
        rows_p = lay[4]
        launch.dk_acc = workspace[lay[6]: lay[6] + 8 * H_KV * rows_p * D].view(torch.int64).view(H_KV, rows_p, D)
        wide = lay[8] == 64
        launch.dv_acc = workspace[lay[7]: lay[7] + (8 if wide else 4) * H_KV * rows_p * D].view(
            torch.int64 if wide else torch.int32).view(H_KV, rows_p, D)
    return launch


def attention_forward(q, k, v, *, causal, softmax_scale=None, cu_seqlens=None, max_seqlen=None, kernel="auto",
                      window=None, sinks=0, o_rest=False):
    """O and LSE (nats) of self-attention through the library's own forward.

    Dense: `(B, S, H, D)` tensors, lse `(B, H, S)`. Varlen: `(total, H, D)`,
    lse `(H, total)`. Stands in for the third-party forward the reference
    calls (src/fold_attention/interface.py:42-44,70-81). `kernel`: "mma" (warp-level,
    every head dim), "sm100" (tcgen05; head_dim 128) or
    "auto". `window` and `sinks` (causal calls): query i sees key j when
    `i - j < window` or `j < sinks`; with `o_rest` such a call returns `(o, lse,
    rest)`, what rounding to 16 bits took from O as 16 bits more, for `prepare_backward`."""
    window, sinks = check_window(window, sinks, causal)
    if o_rest and not window:
        raise ValueError("o_rest is a windowed call's: give a window")
    if kernel not in ("auto", "mma", "sm100"):
        raise ValueError('kernel is one of ("auto", "mma", "sm100")')
    varlen = cu_seqlens is not None
    D = q.shape[-1]
    # the kernels index k and v by q's batch, length and head dim: a mismatch would read past them
    if q.dim() != (3 if varlen else 4) or k.dim() != q.dim() or v.shape != k.shape:
        raise ValueError(f"q is {'(total, H, D)' if varlen else '(B, S, H, D)'}, k and v the same with H_KV heads "
                         f"(got q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)})")
    if k.shape[:-2] != q.shape[:-2] or k.shape[-1] != D or q.shape[-2] % k.shape[-2]:
        raise ValueError(f"k and v {tuple(k.shape)} do not match q {tuple(q.shape)}: same leading sizes and head dim, "
                         "and a head count that divides q's")
    if q.dtype not in (torch.bfloat16, torch.float16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"q, k and v must be bf16 or fp16, and the same type (got {q.dtype}, {k.dtype}, {v.dtype})")
    if any(t.stride(-1) != 1 for t in (q, k, v)) or k.device != q.device or v.device != q.device:
        raise ValueError("q, k and v are on one device with a contiguous head dim")
    if varlen and (cu_seqlens.dtype != torch.int32 or cu_seqlens.device != q.device):
        raise ValueError("cu_seqlens is int32 on q's device")
    sm = float(softmax_scale) if softmax_scale is not None else 1.0 / math.sqrt(D)
    o = torch.empty_like(q)
    rest = torch.empty_like(o) if o_rest else None
    if varlen:
        total, H, _ = q.shape
        B = cu_seqlens.shape[0] - 1
        if max_seqlen is None:
            max_seqlen = int(torch.diff(cu_seqlens).max())
        S = int(max_seqlen)
        lse = torch.empty((H, total), device=q.device, dtype=torch.float32)
        st = []
        for t in (q, k, v, o):
            st += [0, t.stride(0), t.stride(1)]
    else:
        B, S, H, _ = q.shape
        total = B * S
        lse = torch.empty((B, H, S), device=q.device, dtype=torch.float32)
        st = []
        for t in (q, k, v, o):
            st += [t.stride(0), t.stride(1), t.stride(2)]
    strides = (ctypes.c_int64 * 12)(*st)
    can = bool(_lib.lib.fold_fwd_sm100_supported(D, int(q.dtype == torch.float16)))
    if kernel == "sm100" and not can:
        raise NotImplementedError("the tcgen05 forward takes head_dim 128")
    args = [
        q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lse.data_ptr(), ctypes.addressof(strides),
        _lib.ptr(cu_seqlens), B, H, k.shape[-2], S, total, D, int(bool(causal)), int(q.dtype == torch.float16), sm,
    ]
    if can and kernel != "mma":
        status = torch.zeros(1, device=q.device, dtype=torch.int32)
        if window:
            args[5:5] = [_lib.ptr(rest)]
            del args[14]
            with _lib.on(q.device):
                _lib.call("fold_fwd_window_sm100", *args, window, sinks, None, 0, status.data_ptr(), _lib.stream(q.device))
        else:
            _lib.call("fold_fwd_run_sm100", *args, status.data_ptr(), _lib.stream(q.device))
        attention_forward.last_status = status   # non-zero after a device-side wait ran out
        if attention_forward.check_status:
            check_status(status, "attention_forward")
        return (o, lse, rest) if o_rest else (o, lse)
    if window:
        args[5:5] = [_lib.ptr(rest)]
        del args[14]
        with _lib.on(q.device):
            _lib.call("fold_fwd_window", *args, window, sinks, None, 0, _lib.stream(q.device))
    else:
        _lib.call("fold_fwd_run", *args, _lib.stream(q.device))
    return (o, lse, rest) if o_rest else (o, lse)


@functools.lru_cache(maxsize=1024)
def _stride_array(*values):
    """Element strides as the host int64 array a call reads (kept by their values)."""
    return (ctypes.c_int64 * len(values))(*values)


@functools.lru_cache(maxsize=1024)
def _window_workspace(*shape):
    """Bytes of a windowed backward's workspace and its status word's offset, for `(B, H, H_KV, S, total, D, varlen, window, sinks)`."""
    lay = (ctypes.c_int64 * 12)()
    _lib.call("fold_bwd_window_layout", *shape, lay)
    return lay[11], lay[5]


def _packed_strides(ts, varlen):
    """`(batch, row, head)` strides of `(B, S, H, D)` or packed `(total, H, D)` tensors."""
    out = []
    for t in ts:
        st = t.stride()
        out += (0, st[0], st[1]) if varlen else st[:3]
    return _stride_array(*out)


# Delta = dO . O subtracts from dP of the same size where a query sees few keys, and O's rounding to 16 bits then shows
# in dq and dk: 0.0036 of their norm in bf16 where every query sees 2 keys, 0.0026 at 8, 0.0024 from 64 on, against 0.0023 with
# the exact O (the roundings of dS and of the results); what counts is the keys that a row's weight sits on. Up to this
# many visible keys the forward leaves what its rounding took as 16 bits more, and the backward adds it. That is a
# tenth of the time of a large call (16384 tokens of 32 heads, window 128: 606 us without, 664 with; D=64 792 and 875), so
# windows of many keys, whose rows seldom sit on a few of them, go without. The rule knows the window alone: a sequence's bits do
# not depend on what it is packed with, and a larger window that hides nothing is plain causal attention. Sequences of a few
# tokens under a larger window go without too, as they do without a window: 0.0036-0.0039 of dq's and dk's norm in bf16.
REST_KEYS = 256


def window_forward(q, k, v, window, sinks, softmax_scale, cu_seqlens=None, max_seqlen=None, grad=True):
    """`attention_forward` under a window for tensors the public entry points
    have checked: the same kernels with less on the host, which is what a small
    call costs. Returns `(o, lse, o_rest)`; without `grad` no backward follows."""
    varlen = cu_seqlens is not None
    dev, f16 = q.device, int(q.dtype is torch.float16)
    if varlen:
        total, H, D = q.shape
        B, S = cu_seqlens.shape[0] - 1, int(max_seqlen)
        lse = torch.empty((H, total), device=dev, dtype=torch.float32)
    else:
        B, S, H, D = q.shape
        total = B * S
        lse = torch.empty((B, H, S), device=dev, dtype=torch.float32)
    o = torch.empty(q.shape, device=dev, dtype=q.dtype)
    rest = torch.empty_like(o) if grad and window + sinks <= REST_KEYS else None
    strides = _packed_strides((q, k, v, o), varlen)
    args = (q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lse.data_ptr(), _lib.ptr(rest), ctypes.addressof(strides),
            _lib.ptr(cu_seqlens), B, H, k.shape[-2], S, total, D, f16, softmax_scale, window, sinks, None, 0)
    with _lib.on(dev):
        if D == 128 and _lib.lib.fold_fwd_sm100_supported(D, f16):
            status = torch.zeros(1, device=dev, dtype=torch.int32)
            _lib.call("fold_fwd_window_sm100", *args, status.data_ptr(), _lib.stream(dev))
            attention_forward.last_status = status
            if attention_forward.check_status:
                check_status(status, "attention_forward")
        else:
            _lib.call("fold_fwd_window", *args, _lib.stream(dev))
    return o, lse, rest


def window_backward(q, k, v, o, rest, do, lse, window, sinks, softmax_scale, cu_seqlens=None, max_seqlen=None):
    """dQ, dK and dV of `window_forward`'s call, and the status word: what
    `prepare_backward(window=, o_rest=)` launches, once and in the caller's layout."""
    varlen = cu_seqlens is not None
    dev = q.device
    if varlen:
        total, H, D = q.shape
        B, S = cu_seqlens.shape[0] - 1, int(max_seqlen)
    else:
        B, S, H, D = q.shape
        total = B * S
    HKV = k.shape[-2]
    nbytes, at = _window_workspace(B, H, HKV, S, total, D, int(varlen), window, sinks)
    work = torch.empty(nbytes, device=dev, dtype=torch.uint8)
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    strides = _packed_strides((q, k, v, o, do, dq, dk, dv), varlen)
    with _lib.on(dev):
        _lib.call(
            "fold_bwd_window", q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), _lib.ptr(rest), do.data_ptr(), lse.data_ptr(),
            dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), ctypes.addressof(strides), _lib.ptr(cu_seqlens), B, H, HKV, S, total, D,
            int(q.dtype is torch.float16), softmax_scale, work.data_ptr(), nbytes, 0, window, sinks, 15, _lib.stream(dev),
        )
    return dq, dk, dv, work[at:at + 4]


# The tcgen05 forward's status word of the last call; with `check_status` set every call reads
# it back (one host synchronisation per call) and raises FoldLibraryError when it is raised.
attention_forward.last_status = None
attention_forward.check_status = False
