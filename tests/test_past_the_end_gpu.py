"""Captured steps replayed past what a cache has room for: the tokens beyond are dropped, the other requests' planes
keep their bits and their answers stay right, and `sync_lens` tells. Tolerances are test_chunk_gpu's."""

import pytest
import torch

pytestmark = pytest.mark.gpu

from test_chunk_gpu import Story, attend, close, cumulative, make, values_of  # noqa: E402


def captured(call):
    """`call` in a graph of its own, its result and the graph."""
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            out = call()
    return graph, out


def request_want(st, b, q, n):
    """Request b's n newest tokens over all it was brought."""
    return attend(q, *values_of(st.k[b], st.v[b], st.v8, st.evs), st.c.window, st.c.sinks)


@pytest.mark.parametrize("D,page,max_len", [(64, 16, 300), (128, 64, 300), (64, 256, 300), (128, 256, 300)])
@pytest.mark.parametrize("window,sinks", [(60, 3), (None, 0)])
def test_long_chunks_past_the_end_leave_the_others_right(D, page, max_len, window, sinks):
    """Request 0 is at the table's end after two replays; the one behind it in the batch has room throughout."""
    st = Story(2, 8, 2, D, max_len, page_size=page, window=window, sinks=sinks, seed=D)
    st.extend([150, 1])
    new = [120, 33]
    ins = [make(new, h, D, st.dt, st.g) for h in (8, 2, 2)]
    cu = cumulative(new)
    graph, out = captured(lambda: st.c.extend(*ins, cu, new))
    for _ in range(8):
        q, k, v = st.tokens(new)
        for a, b in zip(ins, (q, k, v)):
            a.copy_(b)
        graph.replay()
        close(out[120:], request_want(st, 1, q[120:], 33), st.dt)
    with pytest.raises(ValueError, match=f"max_len={max_len}"):
        st.c.sync_lens()


def pool(c):
    return [t.view(torch.uint8).view(t.shape[0], -1).clone() for t in (c.ka, c.kb, c.va, c.vb, c.ek) if t is not None]


def rows_of(c, b, pos):
    """Pool rows of request b's token at `pos`, one a KV head."""
    page = c.page_table[b, pos // c.page_size].item()
    return [(page * c.n_kv_heads + h) * c.page_size + pos % c.page_size for h in range(c.n_kv_heads)]


def unchanged_but(before, after, rows):
    keep = torch.ones(before[0].shape[0], dtype=torch.bool, device="cuda")
    keep[rows] = False
    return all(torch.equal(a[keep], b[keep]) for a, b in zip(before, after))


@pytest.mark.parametrize("D,page,v8,kw", [
    (64, 16, False, {}), (128, 128, False, dict(kernel="sm100")), (128, 128, True, dict(kernel="sm100", chunk=128)), (128, 64, True, dict(kernel="mma", split=3)),
    (128, 64, False, dict(window=50, sinks=2)), (64, 64, False, dict(depth=12.0, tail=16)),
])
@pytest.mark.parametrize("victim", [0, 2])
def test_one_token_steps_past_the_end_touch_nothing(D, page, v8, kw, victim):
    """The request that runs past the table is the first, whose row another's follows, or the last, whose row nothing follows."""
    B, max_len = 3, 2 * page
    st = Story(B, 8, 2, D, max_len, page_size=page, v8=v8, seed=7, garbage=False, **kw)
    lens = [max_len - 2 if b == victim else 5 + 9 * b for b in range(B)]
    q, k, v = st.tokens(lens)
    st.c.write_prompt(k, v, cumulative(lens), lens)
    assert st.c.v_scale == st.evs          # (the prompt left it on the device: a capture cannot wait for it)
    ins = [make([1] * B, h, D, st.dt, st.g) for h in (8, 2, 2)]
    graph, out = captured(lambda: st.c.decode(*ins))
    others = [b for b in range(B) if b != victim]
    for step in range(6):
        q, k, v = st.tokens([1] * B)
        for a, b in zip(ins, (q, k, v)):
            a.copy_(b)
        before, sums = pool(st.c), st.c.vsum.clone()
        graph.replay()
        may = [r for b in range(B) if lens[b] + step < max_len for r in rows_of(st.c, b, lens[b] + step)]
        assert unchanged_but(before, pool(st.c), may), step
        if "depth" not in kw:       # (a truncating cache drops small weights, by its depth)
            for b in others:
                close(out[b:b + 1], request_want(st, b, q[b:b + 1], 1), st.dt, (step, b))
        if step >= 2:
            mine = slice(victim * 2, victim * 2 + 2)
            assert torch.equal(st.c.vsum[mine], sums[mine]) and torch.isfinite(out).all()
    with pytest.raises(ValueError, match=f"max_len={max_len}"):
        st.c.sync_lens()


@pytest.mark.parametrize("D,page,v8,kw", [
    (64, 16, False, {}), (64, 64, False, {}), (128, 128, True, dict(kernel="sm100")), (128, 64, False, dict(window=50, sinks=2)), (128, 64, True, {}),
    (64, 64, False, dict(depth=12.0, tail=16)),
])
@pytest.mark.parametrize("new", [1, 5, 40])
@pytest.mark.parametrize("victim", [0, 2])
def test_a_pool_that_runs_out_takes_no_page_of_another_request(D, page, v8, kw, new, victim):
    """The victim has two tokens' room when the pool's pages are all in use, and its row of the table named a
    third page for an earlier prompt. New tokens come one a call (a decode step) or several (of which some have a place)."""
    if new > 1 and "tail" in kw:
        pytest.skip("a cache with a tail takes one token at a time")
    if new > 32 and page == 16:
        pytest.skip("the host sees that three pages more do not fit, and refuses")
    B = 3
    st = Story(B, 8, 2, D, 8 * page, page_size=page, v8=v8, seed=3, garbage=False, pages=5, **kw)
    held, lens = 2 * page, [0] * B
    first = [3 * page if b == victim else 1 for b in range(B)]
    st.c.write_prompt(*(make(first, 2, D, st.dt, st.g) for _ in range(2)), cumulative(first), first)
    others = [b for b in range(B) if b != victim]
    lens[victim], lens[others[0]], lens[others[1]] = held - 2, page + 3, 5
    q, k, v = st.tokens(lens)
    st.c.write_prompt(k, v, cumulative(lens), lens)
    assert st.c.v_scale == st.evs and st.c.taken.tolist() == [5]
    news = [new if b == victim else 1 for b in range(B)]
    at = [sum(news[:b]) for b in range(B)]
    ins = [make(news, h, D, st.dt, st.g) for h in (8, 2, 2)]
    cu = cumulative(news)
    st.c.lens[victim] = 0          # (as if captured on a shorter request: the host, which counts pages, refuses one it knows will not fit)
    graph, out = captured(lambda: st.c.decode(*ins) if new == 1 else st.c.extend(*ins, cu, news))
    for step in range(6):
        q, k, v = st.tokens(news)
        for a, b in zip(ins, (q, k, v)):
            a.copy_(b)
        before = pool(st.c)
        graph.replay()
        assert st.c.seq_lens[victim].item() == min(held, lens[victim] + (step + 1) * new)
        may = [r for b in others for r in rows_of(st.c, b, lens[b] + step)]
        for pos in range(lens[victim] + step * new, min(held, lens[victim] + (step + 1) * new)):
            may += rows_of(st.c, victim, pos)
        assert unchanged_but(before, pool(st.c), may), step
        if "depth" not in kw:
            for b in others:
                close(out[at[b]:at[b] + 1], request_want(st, b, q[at[b]:at[b] + 1], 1), st.dt, (step, b))
        assert torch.isfinite(out).all()
    assert (st.c.page_table[victim, :2] >= 0).all() and (st.c.page_table[victim, 2:] == -1).all()
    with pytest.raises(ValueError, match="the pool has 5"):
        st.c.sync_lens()
    # new prompts have the whole pool again
    k, v = (make([page, 1, 2], 2, D, st.dt, st.g) for _ in range(2))
    st.c.write_prompt(k, v, cumulative([page, 1, 2]), [page, 1, 2])
    st.c.sync_lens()
    assert st.c.lens == [page, 1, 2] and st.c.taken.tolist() == [3]


def test_a_pools_table_names_no_page_before_one_is_given():
    import fold_attention_b200 as fa

    c = fa.FoldKVCache(2, 4, 2, 64, 64, page_size=16, pages=5)
    assert (c.page_table == -1).all()
    k = make([20, 3], 2, 64, torch.bfloat16, torch.Generator(device="cuda").manual_seed(0))
    c.append_chunk(k, k, cumulative([20, 3]), [20, 3])
    assert c.page_table.tolist() == [[0, 1, -1, -1], [2, -1, -1, -1]]


def test_a_chunks_sums_count_the_tokens_that_found_a_place():
    """Lengths past a missing page stop there, lengths past the table move on; whole numbers, so sums are exact."""
    from fold_attention_b200.decode import tokens

    dev32 = lambda x: torch.tensor(x, device="cuda", dtype=torch.int32)  # noqa: E731
    n, room = [4, 3, 0, 5], 32
    v = torch.arange(1, 13, device="cuda", dtype=torch.bfloat16)[:, None, None].expand(12, 2, 64).contiguous()
    slots = dev32([7, 8, -1, -1, 3, 4, 5, 20, 21, 22, -1, -1])
    old, new = [14, 2, 9, 29], [18, 5, 9, 34]                         # the third request brings nothing, the last runs past the table
    lens, vsum, vmean = dev32(old), torch.ones(8, 64, device="cuda"), torch.zeros(8, 64, device="cuda")
    tokens.chunk_sums(v, cumulative(n), slots, room, dev32(new), lens, 1.0, vsum, vmean)
    assert lens.tolist() == [16, 5, 9, 34]
    want = [1 + 1 + 2, 1 + 5 + 6 + 7, 1, 1 + 8 + 9 + 10]
    assert vsum.view(4, 2, 64).eq(torch.tensor(want, device="cuda").view(4, 1, 1)).all()
    keys = torch.tensor([16.0, 5.0, 1.0, 32.0], device="cuda")
    mean = torch.tensor(want, device="cuda").float() / keys
    mean[2] = 0
    assert vmean.view(4, 2, 64).eq(mean.view(4, 1, 1)).all()
