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
