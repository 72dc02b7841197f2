"""The windowed forward and backward at the kernel level, with the forward's remainder of O: the public call's bits."""

import pytest
import torch

pytestmark = pytest.mark.gpu

from test_window_gpu import inputs, run_dense, run_packed  # noqa: E402


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,window,sinks", [(128, 2, 0), (128, 100, 4), (96, 3, 1), (64, 256, 0)])
def test_the_pair_gives_the_public_calls_gradients(D, window, sinks, dtype):
    from fold_attention_b200.backward import attention_forward, prepare_backward

    q, k, v, do = (t[None] for t in inputs(500, 4, 2, D, dtype, seed=3))
    want = run_dense(q, k, v, do, window, sinks)
    tr = lambda x: x.transpose(1, 2)  # noqa: E731
    o, lse, rest = attention_forward(q, k, v, causal=True, window=window, sinks=sinks, o_rest=True)
    run = prepare_backward(tr(q), tr(k), tr(v), tr(o), tr(do), lse, causal=True, window=window, sinks=sinks, o_rest=tr(rest))
    assert all(torch.equal(a, b) for a, b in zip((o, *(tr(x) for x in run())), want))
    lens = [300, 1, 199]
    cu = torch.tensor([0, 300, 301, 500], device="cuda", dtype=torch.int32)
    q, k, v, do = (t[0] for t in (q, k, v, do))
    want = run_packed(q, k, v, do, lens, window, sinks)
    kw = dict(causal=True, window=window, sinks=sinks, cu_seqlens=cu, max_seqlen=300)
    o, lse, rest = attention_forward(q, k, v, o_rest=True, **kw)
    assert all(torch.equal(a, b) for a, b in zip((o, *prepare_backward(q, k, v, o, do, lse, o_rest=rest, **kw)()), want))


def test_a_remainder_that_does_not_fit_is_refused():
    from fold_attention_b200.backward import attention_forward, prepare_backward

    q, k, v, do = (t[None] for t in inputs(100, 4, 2, 64, torch.bfloat16, seed=3))
    with pytest.raises(ValueError, match="give a window"):
        attention_forward(q, k, v, causal=True, o_rest=True)
    o, lse, rest = attention_forward(q, k, v, causal=True, window=3, o_rest=True)
    args = [x.transpose(1, 2) for x in (q, k, v, o, do)]
    rest = rest.transpose(1, 2)
    with pytest.raises(ValueError, match="give a window"):
        prepare_backward(*args, lse, causal=True, o_rest=rest)
    for bad in (rest[:, :2], rest.contiguous(), rest.half(), rest.cpu()):
        with pytest.raises(ValueError, match="laid out as o"):
            prepare_backward(*args, lse, causal=True, window=3, o_rest=bad)


@pytest.mark.parametrize("window", [None, 30])
def test_strided_cumulative_lengths_are_the_sequences_they_say(window):
    import fold_attention_b200 as fa

    q, k, v, do = inputs(300, 4, 2, 64, torch.bfloat16, seed=5)
    cu = torch.tensor([0, 9, 120, 9, 300, 9], device="cuda", dtype=torch.int32)[::2]

    def run(cu):
        x = [t.detach().clone().requires_grad_() for t in (q, k, v)]
        out = fa.fold_attn_varlen_func(*x, cu, max_seqlen_q=180, causal=True, window=window)
        return (out.detach(), *torch.autograd.grad(out, x, do))

    want = run(torch.tensor([0, 120, 300], device="cuda", dtype=torch.int32))
    assert all(torch.equal(a, b) for a, b in zip(run(cu), want))
