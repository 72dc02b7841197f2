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
