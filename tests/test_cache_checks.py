"""What a cache refuses, it refuses before it takes a page, moves a length or writes a key."""

import pytest
import torch

import fold_attention_b200 as fa

BF = torch.bfloat16


def cache(**kw):
    """A cache on the CPU, whose kernels cannot run: a call that is not refused first fails in another way."""
    return fa.FoldKVCache(2, 4, 2, 64, 96, page_size=16, device="cpu", **kw)


def state(c):
    return list(c.lens), c.seq_lens.tolist(), c.page_table.tolist(), None if c.taken is None else c.taken.tolist()


@pytest.mark.parametrize("kw", [{}, dict(pages=7), dict(pages=7, window=8), dict(pages=7, depth=9.0, tail=None)])
def test_a_refused_step_leaves_the_cache_as_it_was(kw):
    c = cache(**kw)
    before = state(c)       # empty: the first token of each request would take a page
    q, k = torch.zeros(2, 4, 64, dtype=BF), torch.zeros(2, 2, 64, dtype=BF)
    for bk, bv in ((k[:1], k), (k, k[:, :1]), (k[..., :32], k[..., :32]), (k, k.half()), (k.float(), k.float()), (k.to("meta"), k)):
        with pytest.raises(ValueError, match="k and v|same type|is on"):
            c.append(bk, bv)
        with pytest.raises(ValueError, match="k and v|same type|is on"):
            c.decode(q, bk, bv)
    for bq in (q[:1], q[:, :2], q[..., :32], q.float(), q.to("meta")):
        with pytest.raises(ValueError, match="q is|same type"):
            c.decode(bq, k, k)
    assert state(c) == before


@pytest.mark.parametrize("kw", [{}, dict(pages=7), dict(pages=7, v8=True), dict(pages=7, window=8)])
def test_a_refused_prompt_leaves_the_cache_as_it_was(kw):
    c = cache(**kw)
    before = state(c)
    k, cu = torch.zeros(5, 2, 64, dtype=BF), torch.tensor([0, 3, 5], dtype=torch.int32)
    for bk, bv, lens, match in (
        (k, k[:4], [3, 2], "k and v"), (k, k[..., :32], [3, 2], "k and v"), (k[:, :1], k[:, :1], [3, 2], "k and v"),
        (k.flatten(), k.flatten(), [3, 2], "k and v"), (k, k.half(), [3, 2], "bf16 or fp16"), (k.float(), k.float(), [3, 2], "bf16 or fp16"),
        (k, k, [3, 3], "lens sum to 6"), (k, k, [5], "batch of 2"), (k, k, [5, 0], "not in 1..96"), (k, k, [97, 1], "not in 1..96"),
        (k.to("meta"), k, [3, 2], "k and v are on"),
    ):
        with pytest.raises(ValueError, match=match):
            c.write_prompt(bk, bv, cu, lens)
    if c.taken is not None:
        long = torch.zeros(120, 2, 64, dtype=BF)
        with pytest.raises(ValueError, match="pool has 7"):
            c.write_prompt(long, long, cu, [60, 60])
    assert state(c) == before


def test_an_8_bit_scale_that_chunks_set():
    from fold_attention_b200.decode.write import v_scale_for

    v = torch.tensor([[1.0, -3.5, float("nan")]], dtype=BF)
    assert v_scale_for(v, 2.0) == 2.0 ** -6                       # 7 / 448 is a power of two itself
    assert v_scale_for(v * 1.01, 2.0) == 2.0 ** -5
    assert v_scale_for(v * 0, 2.0) is None
    with pytest.raises(ValueError, match="infinity"):
        v_scale_for(v * float("inf"), 2.0)


def test_a_windowed_cache_refuses_the_splits_it_would_not_keep():
    for kw in (dict(split=2), dict(chunk=64)):
        with pytest.raises(NotImplementedError, match="windowed"):
            cache(window=8, **kw)
    c, q, k = cache(window=8), torch.zeros(2, 4, 64, dtype=BF), torch.zeros(2, 2, 64, dtype=BF)
    for call in (lambda: c.attend(q, split=2), lambda: c.decode(q, k, k, split=2)):
        with pytest.raises(NotImplementedError, match="windowed"):
            call()
    assert state(c)[0] == [0, 0]


@pytest.mark.parametrize("kw", [dict(window=8), dict(pages=7)])
def test_a_caches_writes_run_on_its_own_device(kw, monkeypatch):
    """Whatever the current one is: each launch happens inside `_lib.on` of the cache's device (faked, as is the launch)."""
    import contextlib

    from fold_attention_b200 import _lib

    inside, seen = [], []

    @contextlib.contextmanager
    def on(device):
        inside.append(device)
        yield
        inside.pop()

    monkeypatch.setattr(_lib, "on", on)
    monkeypatch.setattr(_lib, "call", lambda name, *a: seen.append((name, list(inside))))
    monkeypatch.setattr(_lib, "stream", lambda device: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    c, k = cache(**kw), torch.zeros(2, 2, 64, dtype=BF)
    cu = torch.tensor([0, 1, 2], dtype=torch.int32)
    c.write_prompt(k, k, cu, [1, 1])
    c._v_scale = 1.0               # (nothing ran: there is no scale to read)
    c.append(k, k)
    c.append_chunk(k, k, cu, [1, 1])
    assert {"fold_cache_write_prompt", "fold_step_append", "fold_write_tokens", "fold_chunk_sums_placed"} <= {n for n, _ in seen}
    assert all(where == [torch.device("cpu")] for _, where in seen), seen


def test_strided_cumulative_lengths_are_refused():
    """Every other entry of a longer list: the kernels would read the ones between."""
    c, k, q = cache(), torch.zeros(2, 2, 64, dtype=BF), torch.zeros(2, 4, 64, dtype=BF)
    cu = torch.tensor([0, 7, 1, 7, 2, 7], dtype=torch.int32)[::2]
    c.lens = [1, 1]
    for call in (lambda: c.append_chunk(k, k, cu, [1, 1]), lambda: c.attend_chunk(q, cu, [1, 1]), lambda: c.extend(q, k, k, cu, [1, 1])):
        with pytest.raises(ValueError, match="contiguous"):
            call()
