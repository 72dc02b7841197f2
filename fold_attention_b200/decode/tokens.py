"""The paged cache a piece at a time (host side): block tables and slots from
request lengths, new tokens into the pool and back, and the attention of a
chunk of new tokens over the cache that holds them.

A token's slot is `page * page_size + offset`: the same for every KV head, and
for every layer whose cache shares the table, so one `build_tables` serves a
whole model's step. Its pool row for KV head h is
`(page * n_kv_heads + h) * page_size + offset`. A slot of -1 stands for no place:
`write_tokens` skips it and `read_tokens` returns zeros.

No counterpart in the reference, whose tables are the host's and whose cache
takes prompts whole and then one token a request.
"""

from __future__ import annotations

import ctypes
import functools
import math

import torch

from .. import _lib

P, I, F, L = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_int64
_lib.register("fold_build_tables", [P, P, I, P, I, I, I, P, I, P, P, P, P, P])
_lib.register("fold_write_tokens", [P, P, I, L, L, L, L, P, L, I, I, I, L, P, P, P, P, P, F, P])
_lib.register("fold_read_tokens", [P, L, I, I, I, L, P, P, P, P, P, F, P, P, I, P])
_lib.register("fold_chunk_sums", [P, I, L, L, I, I, I, P, I, P, P, F, P, P, P])
_lib.register("fold_chunk_sums_placed", [P, I, L, L, I, I, I, P, I, P, L, P, P, F, P, P, P])
_lib.register("fold_chunk_gather", [P, P, I, P, I, I, I, I, I, I, P, P, P, P, P, F, I, I, I, I, P, P, P, P, P, P])
_lib.register("fold_chunk_sm100", [P, L, L, P, L, L, I, P, P, I, I, I, I, I, P, I, I, L, P, P, P, P, P, F, I, I, I, I, P, L, P, P])
_lib.register("fold_chunk_workspace_bytes", [I, I, I, I, I, I], L)

_HALF = (torch.bfloat16, torch.float16)
_OUT = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _int32(name, t, shape, device):
    if t.dtype is not torch.int32 or t.shape != shape or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} is a contiguous int32 {tuple(shape)} on {device} (got {t.dtype} {tuple(t.shape)} on {t.device})")


def build_tables(cu_seqlens, seq_lens, page_table, page_size, total, *, free_pages=None, taken=None):
    """Block tables and the new tokens' slots, on the device, from lengths.

    Request b holds `seq_lens[b]` tokens and brings rows `cu_seqlens[b] ..
    cu_seqlens[b + 1]` of `total` packed ones (none is allowed). With
    `free_pages`, an int32 list of page numbers whose first `taken[0]` are in
    use, the pages a request grows by are taken from it in request order and
    written into `page_table` `(batch, pages)`, in place; without, the table
    stands as it is. Returns `(slots, lens, taken)`: each new token's slot
    (int32 `(total,)`), the lengths with the new tokens, and the pages then in
    use (None without `free_pages`). A token that its request's table row or
    the pool has no page for, or whose page in the table is negative, and a row
    that no request covers, gets slot -1; `taken` past the list's end says that
    the pool ran out. The entry of a page that the pool could not give stands as
    it was, and calls on the longer lengths read it: a table over a pool that may
    run out starts as -1 throughout. The arguments other
    than the table are left as they are, so the same call gives the same
    answer. All tensors are int32 on one device; nothing waits on it.
    """
    total, page_size = int(total), int(page_size)
    B = seq_lens.numel()
    if not (seq_lens.dtype is cu_seqlens.dtype is page_table.dtype is torch.int32 and seq_lens.ndim == 1 and page_table.ndim == 2
            and cu_seqlens.shape == (B + 1,) and page_table.shape[0] == B and seq_lens.is_contiguous() and cu_seqlens.is_contiguous()
            and page_table.is_contiguous() and cu_seqlens.get_device() == page_table.get_device() == seq_lens.get_device()
            and B > 0 and page_table.shape[1] > 0):
        _tables_refused(cu_seqlens, seq_lens, page_table)
    if total < 0 or page_size < 1:
        raise ValueError(f"{total} tokens, pages of {page_size} keys")
    if (free_pages is None) != (taken is None):
        raise ValueError("free_pages and taken are both given or both left out")
    dev = seq_lens.device
    n_free, used = 0, None
    if free_pages is not None:
        n_free = free_pages.numel()
        _int32("free_pages", free_pages, (n_free,), dev)
        _int32("taken", taken, (1,), dev)
        used = torch.empty_like(taken)
    slots, lens = seq_lens.new_empty(total), torch.empty_like(seq_lens)
    with _lib.on(dev):
        _lib.call(
            "fold_build_tables", cu_seqlens.data_ptr(), seq_lens.data_ptr(), B, page_table.data_ptr(), page_table.shape[1], page_size,
            total, _lib.ptr(free_pages) or None, n_free, _lib.ptr(taken), slots.data_ptr(), lens.data_ptr(), _lib.ptr(used), _lib.stream(dev),
        )
    return slots, lens, used


def _tables_refused(cu_seqlens, seq_lens, page_table):
    dev, B = seq_lens.device, seq_lens.numel()
    if seq_lens.ndim != 1 or page_table.ndim != 2 or B < 1 or page_table.shape[1] < 1:
        raise ValueError(f"seq_lens is (batch,) and page_table (batch, pages), got {tuple(seq_lens.shape)}, {tuple(page_table.shape)}")
    _int32("seq_lens", seq_lens, (B,), dev)
    _int32("cu_seqlens", cu_seqlens, (B + 1,), dev)
    _int32("page_table", page_table, (B, page_table.shape[1]), dev)


def _planes(D, ka, kb, va, vb, ek, dev):
    """The pool's planes, checked against each other: the kernels index all of them by one row."""
    shape = (ka.shape[0], D)
    ok = (ka.dtype is kb.dtype is torch.int8 and ek.dtype is torch.bfloat16 and ka.shape == kb.shape == va.shape == shape
          and ek.shape == shape[:1] and ka.device == dev and kb.get_device() == va.get_device() == ek.get_device() == ka.get_device()
          and ka.is_contiguous() and kb.is_contiguous() and va.is_contiguous() and ek.is_contiguous())
    if vb is None:
        ok = ok and va.dtype is torch.bfloat16
    else:
        ok = (ok and va.dtype is vb.dtype is torch.float8_e4m3fn and vb.shape == shape and vb.get_device() == ka.get_device()
              and vb.is_contiguous())
    if ok:
        return
    vdt = torch.bfloat16 if vb is None else torch.float8_e4m3fn
    for name, t, dt, want in (("ka", ka, torch.int8, shape), ("kb", kb, torch.int8, shape), ("va", va, vdt, shape),
                              ("vb", vb, vdt, shape), ("ek", ek, torch.bfloat16, shape[:1])):
        if t is not None and (t.dtype is not dt or t.shape != want or t.device != dev or not t.is_contiguous()):
            raise ValueError(f"{name} is a contiguous {dt} {want} on {dev} (got {t.dtype} {tuple(t.shape)} on {t.device})")


def _rows(t):
    """`t` with 16-byte rows the kernels can read in place, or a copy."""
    a, b, c = t.stride()
    return t if c == 1 and not (a | b) & 7 and not t.data_ptr() & 15 else t.clone(memory_format=torch.contiguous_format)


def write_tokens(k, v, slots, page_size, ka, kb, va, vb, ek, *, v_scale=1.0):
    """Quantise `k`, `v` `(total, H_KV, D)` (bf16 or fp16) into the pool at
    `slots`: the planes a prompt's write or a step's append puts there. `vb`
    None is a bf16 V; `v_scale` is an 8-bit V's power of two. The slots are
    distinct (two tokens of one call in one slot would leave a mixture); a
    token whose slot is negative or beyond the pool is skipped."""
    if k.ndim != 3 or v.shape != k.shape or k.dtype not in _HALF or v.dtype != k.dtype:
        raise ValueError(f"k and v are (total, H_KV, D) of one 16-bit type (got {k.dtype} {tuple(k.shape)}, {v.dtype} {tuple(v.shape)})")
    n, HKV, D = k.shape
    dev = k.device
    if D not in (64, 128):
        raise NotImplementedError(f"head_dim {D}: the cache takes 64 or 128")
    if v.device != dev:
        raise ValueError(f"k is on {dev}, v on {v.device}")
    _int32("slots", slots, (n,), dev)
    _planes(D, ka, kb, va, vb, ek, dev)
    k, v = _rows(k), _rows(v)
    k0, k1, _ = k.stride()
    v0, v1, _ = v.stride()
    with _lib.on(dev):
        _lib.call(
            "fold_write_tokens", k.data_ptr(), v.data_ptr(), int(k.dtype is torch.float16), k0, k1, v0, v1,
            slots.data_ptr(), n, HKV, D, int(page_size), ka.shape[0], ka.data_ptr(), kb.data_ptr(), va.data_ptr(), _lib.ptr(vb),
            ek.data_ptr(), float(v_scale), _lib.stream(dev),
        )


def read_tokens(slots, page_size, n_kv_heads, ka, kb, va, vb, ek, *, v_scale=1.0, dtype=torch.bfloat16):
    """The tokens at `slots` as the values their codes stand for: `(k, v)`, each
    `(total, H_KV, D)` in `dtype` (float32, bfloat16 or float16, which
    saturates), keys in their own basis. Slots may repeat; zeros at a slot that
    is negative or beyond the pool."""
    if dtype not in _OUT:
        raise ValueError(f"dtype is float32, bfloat16 or float16 (got {dtype})")
    dev, D = ka.device, ka.shape[-1]
    if D not in (64, 128):
        raise NotImplementedError(f"head_dim {D}: the cache takes 64 or 128")
    n, HKV = slots.shape[0], int(n_kv_heads)
    _int32("slots", slots, (n,), dev)
    _planes(D, ka, kb, va, vb, ek, dev)
    k = ka.new_empty((n, HKV, D), dtype=dtype)
    v = torch.empty_like(k)
    with _lib.on(dev):
        _lib.call(
            "fold_read_tokens", slots.data_ptr(), n, HKV, D, int(page_size), ka.shape[0], ka.data_ptr(), kb.data_ptr(), va.data_ptr(), _lib.ptr(vb),
            ek.data_ptr(), float(v_scale), k.data_ptr(), v.data_ptr(), _OUT[dtype], _lib.stream(dev),
        )
    return k, v


def chunk_sums(v, cu_seqlens, slots, room, lens_new, seq_lens, v_scale, vsum, vmean):
    """The running V sums and means with a chunk's `v` added, and `seq_lens` set to `lens_new`: of the tokens
    whose `slots` are a place, and up to the first page that is missing of the `room` keys in the table."""
    n, HKV, D = v.shape
    v = _rows(v)
    with _lib.on(v.device):
        _lib.call(
            "fold_chunk_sums_placed", v.data_ptr(), int(v.dtype == torch.float16), v.stride(0), v.stride(1), seq_lens.shape[0], HKV, D,
            cu_seqlens.data_ptr(), n, slots.data_ptr(), room, lens_new.data_ptr(), seq_lens.data_ptr(), float(v_scale), vsum.data_ptr(), vmean.data_ptr(),
            _lib.stream(v.device),
        )


@functools.lru_cache(maxsize=None)
def _sms(index):
    return torch.cuda.get_device_properties(index).multi_processor_count


SHORT_ROWS = 128     # new tokens x query heads a KV head that chunk_sm100.cu takes


# Where a batch holds wider requests too, its short ones get the second kernel only if that many 128-key tiles
# (x KV heads) pay for it: nine requests of up to 1500 keys and two KV heads take 57 us dequantised together and 97 with
# both kernels; a decode batch's long contexts read from the codes at a third of the bytes. It is a rule on the batch: a short
# request's keys are exact from the codes in one batch and rounded to q's 16 bits in another.
MIXED_TILES = 1024


def chunk_attention(q, cu_seqlens, lens, cap_tiles, seq_lens, page_table, page_size, ka, kb, va, vb, ek, v_scale, n_kv_heads,
                    window, sinks):
    """Attention of each request's last tokens over the pool: `q` `(total, H,
    D)`, cut by `cu_seqlens`, `lens[b]` rows of request b. `cap_tiles` is two
    counts of 128-key tiles at most: of the requests with up to `SHORT_ROWS` query
    rows a KV head, which are attended straight from the codes, and of the
    others, whose keys are dequantised first. Returns `(out, status)`."""
    total, H, D = q.shape
    dev, dt = q.device, q.dtype
    B, G = seq_lens.shape[0], H // n_kv_heads
    f16, win = int(dt == torch.float16), window or 1 << 30
    short, wide = cap_tiles[0] > 0, cap_tiles[1] > 0
    if short and wide and cap_tiles[0] * n_kv_heads < MIXED_TILES:
        short, cap_tiles = False, sum(cap_tiles)
    else:
        cap_tiles = cap_tiles[1]
    out = torch.empty((total, H, D), device=dev, dtype=dt)
    n_plan = -(-(5 * B + 1) // 2) * 2      # (the tile map sits on 8 bytes)
    work = torch.empty(4 + (n_plan + 2 * cap_tiles if wide else 0), device=dev, dtype=torch.int32)
    status = work[:1]
    pool = (page_table.data_ptr(), page_table.shape[1], int(page_size))
    planes = (ka.data_ptr(), kb.data_ptr(), va.data_ptr(), _lib.ptr(vb), ek.data_ptr(), float(v_scale))
    base = work.data_ptr()
    with _lib.on(dev):
        st = _lib.stream(dev)
        if short:
            ctas = _sms(dev.index)
            nbytes = _lib.lib.fold_chunk_workspace_bytes(B, total, H, n_kv_heads, D, ctas)
            space = torch.empty(nbytes, device=dev, dtype=torch.uint8)
            _lib.call(
                "fold_chunk_sm100", q.data_ptr(), q.stride(0), q.stride(1), out.data_ptr(), out.stride(0), out.stride(1), f16,
                cu_seqlens.data_ptr(), seq_lens.data_ptr(), B, total, H, n_kv_heads, D, *pool, ka.shape[0], *planes, win, sinks, int(wide),
                ctas, space.data_ptr(), nbytes, base, st,
            )
        if wide:
            rows = cap_tiles * 128
            kw = torch.empty((2, n_kv_heads, rows, D), device=dev, dtype=dt)
            vw = kw.data_ptr() + kw.stride(0) * 2
            plan = base + 16
            _lib.call(
                "fold_chunk_gather", cu_seqlens.data_ptr(), seq_lens.data_ptr(), B, *pool, n_kv_heads, D, win, sinks, *planes, f16,
                SHORT_ROWS if short else 0, G, cap_tiles, plan, plan + 4 * n_plan, kw.data_ptr(), vw, base, st,
            )
            strides = (ctypes.c_int64 * 12)(0, q.stride(0), q.stride(1), 0, D, rows * D, 0, D, rows * D, 0, out.stride(0), out.stride(1))
            args = (q.data_ptr(), kw.data_ptr(), vw, out.data_ptr(), None, None, ctypes.addressof(strides), cu_seqlens.data_ptr(), B, H,
                    n_kv_heads, max(lens), total, D, f16, 1.0 / math.sqrt(D), win, sinks, plan, rows)
            if _lib.lib.fold_fwd_sm100_supported(D, f16):
                _lib.call("fold_fwd_window_sm100", *args, base, st)
            else:
                _lib.call("fold_fwd_window", *args, st)
    return out, status
