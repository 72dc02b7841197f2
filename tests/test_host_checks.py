"""Host-side argument checks that need no GPU: they raise before any launch."""

import pytest
import torch


def _step_args(q, k, v):
    from fold_attention_b200.decode import write

    B, H, HKV, D = 2, 4, 2, 64
    z8 = torch.zeros(8, D, dtype=torch.int8)
    lens = torch.zeros(B, dtype=torch.int32)
    return write.step, (q, k, v, z8, z8, torch.zeros(8), torch.zeros(8, dtype=torch.bfloat16),
                        torch.zeros(B, 1, dtype=torch.int32), 64, lens, z8, z8, z8, None, 1.0,
                        torch.zeros(B * HKV, D), torch.zeros(B * HKV, D), lens)


@pytest.mark.parametrize("qd,kd,vd", [
    (torch.float32, torch.bfloat16, torch.bfloat16),
    (torch.bfloat16, torch.float16, torch.float16),
    (torch.float16, torch.float16, torch.bfloat16),
    (None, torch.float32, torch.float32),
])
def test_a_step_refuses_mixed_or_wide_dtypes(qd, kd, vd):
    """The step kernel reads q, k and v as one 16-bit type (the reference binds its step per
    dtype, src/fold_attention/decode/write.py:565-673): anything else is refused on the host."""
    B, H, HKV, D = 2, 4, 2, 64
    q = None if qd is None else torch.zeros(B * H, D, dtype=qd)
    k, v = torch.zeros(B, HKV, D, dtype=kd), torch.zeros(B, HKV, D, dtype=vd)
    step, args = _step_args(q, k, v)
    with pytest.raises(ValueError, match="must be bf16 or fp16"):
        step(*args)


def test_status_text():
    from fold_attention_b200 import _lib
    from fold_attention_b200.utils import check_status

    check_status(None, "x")
    check_status(torch.zeros(1, dtype=torch.int32), "x")
    with pytest.raises(_lib.FoldLibraryError, match="x: a device-side wait ran out"):
        check_status(torch.tensor([3], dtype=torch.int32), "x")
    with pytest.raises(_lib.FoldLibraryError, match="refused its arguments"):
        check_status(torch.tensor([1], dtype=torch.int32), "x")


def test_the_forward_and_backward_refuse_tensors_that_do_not_match_q():
    """The kernels index k, v, o, do and lse by q's sizes, so a mismatch is refused on the host
    (CPU tensors here: the checks come before any launch)."""
    from fold_attention_b200.backward.launch import attention_forward, prepare_backward

    B, S, H, HKV, D = 2, 16, 4, 2, 64
    q = torch.zeros(B, S, H, D, dtype=torch.bfloat16)
    k = torch.zeros(B, S, HKV, D, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="do not match q"):
        attention_forward(q, k[:, :8], k[:, :8], causal=True)          # a shorter k: would be read past its end
    with pytest.raises(ValueError, match="do not match q"):
        attention_forward(q.transpose(1, 2), k, k, causal=True)        # (B, H, S, D) passed where (B, S, H, D) goes
    with pytest.raises(ValueError, match="H_KV heads"):
        attention_forward(q, k, k[:, :, :1], causal=True)
    with pytest.raises(ValueError, match="same type"):
        attention_forward(q, k.half(), k.half(), causal=True)
    with pytest.raises(ValueError, match="contiguous head dim"):
        attention_forward(q.transpose(-1, -2).contiguous().transpose(-1, -2), k, k, causal=True)
    with pytest.raises(ValueError, match="int32"):
        attention_forward(q[0], k[0], k[0], causal=True, cu_seqlens=torch.tensor([0, 16]), max_seqlen=16)

    qb, kb = q.transpose(1, 2), k.transpose(1, 2)                      # the backward's (B, H, S, D) views
    lse = torch.zeros(B, H, S)
    with pytest.raises(ValueError, match="do not match q"):
        prepare_backward(qb, kb[:1], kb[:1], qb, qb, lse, causal=True)
    with pytest.raises(ValueError, match="o and do are q's shape"):
        prepare_backward(qb, kb, kb, qb[:, :2], qb, lse, causal=True)
    with pytest.raises(ValueError, match=r"lse is \(B, H, S\)"):
        prepare_backward(qb, kb, kb, qb, qb, lse[:, :, :8], causal=True)
    with pytest.raises(ValueError, match="same 16-bit type"):
        prepare_backward(qb, kb, kb, qb.half(), qb, lse, causal=True)
    with pytest.raises(NotImplementedError, match="self-attention"):
        prepare_backward(qb, kb[:, :, :8], kb[:, :, :8], qb, qb, lse, causal=True)


def test_a_decode_launch_binds_on_the_host_for_every_layout():
    """`prepare_fold_decode` validates and binds without touching the GPU: every layout it takes
    builds a launch from CPU tensors (nothing is run), and the mismatches are refused."""
    from fold_attention_b200.decode.launch import prepare_fold_decode

    def planes(NBH, G, D=128):
        return (torch.zeros(NBH, G, D, dtype=torch.int8), torch.zeros(NBH, G, D, dtype=torch.int8), torch.ones(NBH, G),
                torch.zeros(1024, D, dtype=torch.int8), torch.zeros(1024, D, dtype=torch.int8), torch.zeros(1024, dtype=torch.bfloat16),
                torch.zeros(1024, D, dtype=torch.bfloat16), torch.zeros(NBH, G), torch.full((NBH, G), 8.0))

    kw = dict(page_table=torch.zeros(2, 4, dtype=torch.int32), page_size=64, seq_lens=torch.zeros(2, dtype=torch.int32), n_kv_heads=2)
    assert prepare_fold_decode(*planes(4, 8), truncate=True, vmean=torch.zeros(4, 128), **kw).kernel in ("mma", "sm100")
    assert prepare_fold_decode(*planes(4, 8), truncate=True, vmean=torch.zeros(4, 128), draft_len=4, causal=True, **kw).tree.shape == (4, 8)
    assert prepare_fold_decode(*planes(4, 8), truncate=True, vmean=torch.zeros(4, 8, 128), **kw).kernel == "mma"
    assert prepare_fold_decode(*planes(4, 8), truncate=True, vmean=torch.zeros(4, 128), sound=True, **kw).kernel == "mma"
    assert prepare_fold_decode(*planes(4, 8), truncate=True, vmean=torch.zeros(4, 128), group_cut=False, **kw).kernel == "mma"
    assert prepare_fold_decode(*planes(4, 32), split=2, **kw).kernel == "mma"      # 16 groups of 8 on the warp-level kernel
    with pytest.raises(ValueError, match="one per query row"):
        prepare_fold_decode(*planes(4, 8), truncate=True, vmean=torch.zeros(4, 4, 128), **kw)
    with pytest.raises(NotImplementedError, match="16, 24 or 32"):
        prepare_fold_decode(*planes(4, 12), **kw)
    with pytest.raises(NotImplementedError, match="one group of at most 8"):
        prepare_fold_decode(*planes(4, 16), draft_len=2, causal=True, **kw)
    with pytest.raises(ValueError, match="names the 16 groups of 8"):
        prepare_fold_decode(*planes(4, 32), order=torch.arange(4, dtype=torch.int32), **kw)


@pytest.mark.parametrize("window,sinks,causal", [
    (0, 0, True), (-1, 0, True), (2.5, 0, True), (True, 0, True), (4, -1, True), (4, 1.5, True), (4, 0, False),
    (None, 3, True), ((1 << 30) + 1, 0, True), (4, (1 << 30) + 1, True),
])
def test_a_window_that_means_nothing_is_refused(window, sinks, causal):
    import fold_attention_b200 as fa

    x = torch.zeros(1, 8, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="window"):
        fa.fold_attn_func(x, x, x, causal=causal, window=window, sinks=sinks)
    cu = torch.tensor([0, 8], dtype=torch.int32)
    with pytest.raises(ValueError, match="window"):
        fa.fold_attn_varlen_func(x[0], x[0], x[0], cu, causal=causal, window=window, sinks=sinks)


def test_a_windowed_backward_takes_no_plan():
    from fold_attention_b200.backward import Plan, prepare_backward

    x = torch.zeros(1, 2, 8, 64, dtype=torch.bfloat16)
    with pytest.raises(NotImplementedError, match="plan"):
        prepare_backward(x, x, x, x, x, torch.zeros(1, 2, 8), causal=True, window=4, plan=Plan(1, 0))


def _cpu_cache(**kw):
    import fold_attention_b200 as fa

    return fa.FoldKVCache(2, 4, 2, 64, 96, page_size=16, device="cpu", **kw)


@pytest.mark.parametrize("kw,error,match", [
    (dict(window=0), ValueError, "window"), (dict(sinks=2), ValueError, "window"), (dict(window=8, sinks=-1), ValueError, "window"),
    (dict(window=8, depth=12.0), NotImplementedError, "depth=None"), (dict(pages=0), ValueError, "pool"),
])
def test_a_cache_refuses_windows_and_pools_that_mean_nothing(kw, error, match):
    with pytest.raises(error, match=match):
        _cpu_cache(**kw)


def test_chunks_are_checked_before_anything_is_written():
    bf = torch.bfloat16
    c = _cpu_cache(pages=7)
    cu = torch.tensor([0, 3, 5], dtype=torch.int32)
    q, k = torch.zeros(5, 4, 64, dtype=bf), torch.zeros(5, 2, 64, dtype=bf)
    for bad in (cu.long(), cu[:2]):
        with pytest.raises(ValueError, match="cu_seqlens"):
            c.extend(q, k, k, bad, [3, 2])
    for lens in ([3], [6, -1]):
        with pytest.raises(ValueError, match="counts"):
            c.extend(q, k, k, cu, lens)
    for bad in (q[:4], q.float(), q[:, :2], q[..., :32]):
        with pytest.raises(ValueError, match="q is"):
            c.extend(bad, k, k, cu, [3, 2])
    for bk, bv in ((k[:4], k), (k, k[:, :1]), (k, k.half()), (k.float(), k.float())):
        with pytest.raises(ValueError, match="k and v"):
            c.extend(q, bk, bv, cu, [3, 2])
    with pytest.raises(ValueError, match="more query rows"):
        c.attend_chunk(q, cu, [3, 2])
    long = torch.zeros(97, 2, 64, dtype=bf)
    with pytest.raises(ValueError, match="max_len"):
        c.append_chunk(long, long, torch.tensor([0, 97, 97], dtype=torch.int32), [97, 0])
    with pytest.raises(ValueError, match="pool has 7"):
        c.append_chunk(torch.cat((long, long))[:120], torch.cat((long, long))[:120], torch.tensor([0, 60, 120], dtype=torch.int32), [60, 60])
    assert c.lens == [0, 0]
    t = _cpu_cache(depth=8.0, tail=None)
    assert t.tail is None
    with pytest.raises(ValueError, match="cu_seqlens"):
        import fold_attention_b200 as fa

        fa.fold_attn_with_kvcache(q, c, lens=[3, 2])
    for call in (lambda c: c.prepare_replay_decode(), lambda c: c.tune_split(), lambda c: c.prepare_replay_step(q)):
        with pytest.raises(NotImplementedError, match="windowed"):
            call(_cpu_cache(window=8))


def test_tables_and_tokens_are_checked():
    from fold_attention_b200 import decode

    i32 = torch.int32
    cu, lens, table = torch.zeros(3, dtype=i32), torch.zeros(2, dtype=i32), torch.zeros(2, 4, dtype=i32)
    one = torch.zeros(1, dtype=i32)
    for args, kw in (
        ((cu.long(), lens, table, 16, 0), {}), ((cu[:2], lens, table, 16, 0), {}), ((cu, lens, table.t(), 16, 0), {}),
        ((cu, lens, table, 0, 0), {}), ((cu, lens, table, 16, -1), {}), ((cu, lens, table, 16, 0), dict(free_pages=one)),
        ((cu, lens, table, 16, 0), dict(free_pages=one, taken=torch.zeros(2, dtype=i32))), ((cu, lens[:0], table[:0], 16, 0), {}),
    ):
        with pytest.raises(ValueError):
            decode.build_tables(*args, **kw)
    ka = torch.zeros(32, 64, dtype=torch.int8)
    va, ek = torch.zeros(32, 64, dtype=torch.bfloat16), torch.zeros(32, dtype=torch.bfloat16)
    k, slots = torch.zeros(5, 2, 64, dtype=torch.bfloat16), torch.zeros(5, dtype=i32)
    for bad in (dict(k=k.float()), dict(k=k[:4]), dict(slots=slots.long()), dict(slots=slots[:4]), dict(ka=ka[:16]), dict(va=va.half()),
                dict(ek=ek.float()), dict(vb=va)):
        a = dict(k=k, v=k, slots=slots, page_size=16, ka=ka, kb=ka, va=va, vb=None, ek=ek)
        a.update(bad)
        with pytest.raises(ValueError):
            decode.write_tokens(**a)
    with pytest.raises(NotImplementedError, match="head_dim"):
        decode.write_tokens(k[..., :32], k[..., :32], slots, 16, ka, ka, va, None, ek)
    for bad in (dict(dtype=torch.int8), dict(slots=slots.long()), dict(ka=ka.float()), dict(ek=ek[:8])):
        a = dict(slots=slots, page_size=16, n_kv_heads=2, ka=ka, kb=ka, va=va, vb=None, ek=ek)
        a.update(bad)
        with pytest.raises(ValueError):
            decode.read_tokens(**a)


@pytest.mark.parametrize("plane", range(4))
def test_pool_planes_off_a_16_byte_boundary_are_refused(plane):
    """Before anything is launched: the addresses are never read."""
    from fold_attention_b200 import _lib
    from fold_attention_b200.decode import tokens  # noqa: F401 (declares the entry points)

    planes = [0x1000] * 4
    planes[plane] += 8
    with pytest.raises(ValueError, match="16-byte aligned"):
        _lib.call("fold_write_tokens", 0x1000, 0x1000, 0, 128, 64, 128, 64, 0x1000, 3, 2, 64, 16, 64, *planes, 0x1000, 1.0, None)
    with pytest.raises(ValueError, match="16-byte aligned"):
        _lib.call("fold_read_tokens", 0x1000, 3, 2, 64, 16, 64, *planes, 0x1000, 1.0, 0x1000, 0x1000, 1, None)
    with pytest.raises(ValueError, match="16-byte aligned"):
        _lib.call("fold_chunk_gather", 0x1000, 0x1000, 2, 0x1000, 4, 16, 2, 64, 1 << 30, 0, *planes, 0x1000, 1.0, 0, 0, 2, 4,
                  0x1000, 0x1000, 0x1000, 0x1000, 0x1000, None)
