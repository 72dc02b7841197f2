"""Causal self-attention under a sliding window with sinks: forward, gradients, and what the
backward promises of its bits, against a plain 64-bit implementation.

Tolerances. The forward's P is rounded to 16 bits (relative 2^-9 bf16, 2^-12 fp16 in the root mean
square: half a step is 2^-8 / 2^-11 at worst and uniform below it) and so is O: together under one
half step, 2^-8 / 2^-11, of an output's own size in the root mean square. In the backward P, dS, O (in Delta) and the result
are each rounded once: four roundings, under 2 half steps in the root mean square."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def reference(q, k, v, do, window, sinks):
    """One sequence (n, heads, dim) in 64 bits: out, dq, dk, dv."""
    n, H, D = q.shape
    G = H // k.shape[1]
    a, b, c = (x.double().requires_grad_() for x in (q, k, v))
    i = torch.arange(n, device=q.device)
    seen = (i[None] <= i[:, None]) & ((i[:, None] - i[None] < window) | (i[None] < sinks))
    kk, vv = b.repeat_interleave(G, 1), c.repeat_interleave(G, 1)
    s = torch.einsum("ihd,jhd->hij", a, kk) / math.sqrt(D)
    p = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
    o = torch.einsum("hij,jhd->ihd", p, vv)
    grads = torch.autograd.grad(o, (a, b, c), do.double())
    with torch.no_grad():
        A = (o * do.double()).abs().sum(-1)                                    # (n, H)
        slack_q = torch.einsum("hij,jhd->ihd", p, kk.abs()) * A[..., None] / math.sqrt(D)
        slack_k = torch.einsum("hij,ihd->jhd", p, A[..., None] * a.abs()).view(n, -1, G, D).sum(2) / math.sqrt(D)
    return (o.detach(), *grads, slack_q, slack_k)


def inputs(total, H, HKV, D, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q, do = (torch.randn(total, H, D, device="cuda", generator=g).to(dtype) for _ in range(2))
    k, v = (torch.randn(total, HKV, D, device="cuda", generator=g).to(dtype) for _ in range(2))
    return q, k, v, do


def run_dense(q, k, v, do, window, sinks):
    import fold_attention_b200 as fa

    x = [t.detach().clone().requires_grad_() for t in (q, k, v)]
    out = fa.fold_attn_func(*x, causal=True, window=window, sinks=sinks)
    return (out.detach(), *torch.autograd.grad(out, x, do))


def run_packed(q, k, v, do, lens, window, sinks):
    import fold_attention_b200 as fa

    cu = torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), device="cuda", dtype=torch.int32)
    x = [t.detach().clone().requires_grad_() for t in (q, k, v)]
    out = fa.fold_attn_varlen_func(*x, cu, max_seqlen_q=max(lens), causal=True, window=window, sinks=sinks)
    return (out.detach(), *torch.autograd.grad(out, x, do))


def check(got, want, dtype):
    eps = half_step(dtype)
    slack = {"dq": want[4].norm().item() * eps, "dk": want[5].norm().item() * eps}
    for name, a, b, steps in zip(("out", "dq", "dk", "dv"), got, want, (1, 2, 2, 2)):
        assert torch.isfinite(a).all(), name
        err, tol = (a.double() - b).norm().item(), steps * eps * b.norm().item() + slack.get(name, 0.0)
        assert err <= tol, (name, err, tol)


@pytest.mark.parametrize("S,window,sinks", [
    (1, 1, 0), (1, 5, 3), (2, 1, 1), (63, 7, 2), (127, 128, 4), (128, 1, 0), (129, 127, 1), (256, 128, 128), (257, 129, 129),
    (300, 1, 4), (511, 64, 0), (700, 130, 300), (1037, 77, 5), (1500, 1000, 4), (1281, 3000, 7), (2100, 200, 1),
])
@pytest.mark.parametrize("D", [128, 64])
def test_dense_window_and_gradients(S, window, sinks, D):
    dt = torch.bfloat16
    B, H, HKV = 2, 4, 2
    q, k, v, do = inputs(B * S, H, HKV, D, dt, seed=S)
    got = run_dense(*(x.view(B, S, -1, D) for x in (q, k, v, do)), window, sinks)
    for b in range(B):
        sl = slice(b * S, (b + 1) * S)
        check([g[b] for g in got], reference(q[sl], k[sl], v[sl], do[sl], window, sinks), dt)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D,H,HKV", [(128, 6, 2), (96, 6, 2), (64, 8, 8), (128, 8, 1)])
@pytest.mark.parametrize("window,sinks", [(100, 0), (77, 5), (260, 140)])
def test_packed_window_and_gradients(dtype, D, H, HKV, window, sinks):
    dt = DT[dtype]
    lens = [1, 333, 64, 900, 129]
    q, k, v, do = inputs(sum(lens), H, HKV, D, dt, seed=D + window)
    got = run_packed(q, k, v, do, lens, window, sinks)
    at = 0
    for n in lens:
        sl = slice(at, at + n)
        check([g[sl] for g in got], reference(q[sl], k[sl], v[sl], do[sl], window, sinks), dt)
        at += n


@pytest.mark.parametrize("D", [128, 64])
def test_a_window_no_sequence_fills_is_causal_attention(D):
    import fold_attention_b200 as fa

    q, k, v, do = inputs(2 * 500, 4, 2, D, torch.bfloat16)
    q, k, v, do = (x.view(2, 500, -1, D) for x in (q, k, v, do))
    x = [t.clone().requires_grad_() for t in (q, k, v)]
    out = fa.fold_attn_func(*x, causal=True)
    plain = (out.detach(), *torch.autograd.grad(out, x, do))
    for got, want in zip(run_dense(q, k, v, do, 500, 0), plain):
        assert torch.equal(got, want)
    huge = run_dense(q, k, v, do, 1 << 30, 1 << 30)
    assert torch.equal(huge[0], plain[0]) and torch.equal(huge[1], plain[1])


@pytest.mark.parametrize("D", [128, 96])
def test_bits_do_not_depend_on_the_packing_or_the_run(D):
    lens, window, sinks = [700, 1300, 90, 2000], 150, 9
    q, k, v, do = inputs(sum(lens), 4, 2, D, torch.bfloat16, seed=5)
    first = run_packed(q, k, v, do, lens, window, sinks)
    again = run_packed(q, k, v, do, lens, window, sinks)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    at = 0
    for n in lens:
        sl = slice(at, at + n)
        alone = run_packed(q[sl], k[sl], v[sl], do[sl], [n], window, sinks)
        assert all(torch.equal(a[sl], b) for a, b in zip(first, alone))
        dense = run_dense(*(x[sl][None] for x in (q, k, v, do)), window, sinks)
        assert all(torch.equal(a[sl], b[0]) for a, b in zip(first, dense))
        at += n


def test_gradients_against_differences():
    """The loss's own change along a direction, from the forward in 64 bits, against the kernels' gradients."""
    S, H, HKV, D, window, sinks = 400, 2, 1, 128, 60, 3
    q, k, v, do = inputs(S, H, HKV, D, torch.float16, seed=9)
    got = run_dense(*(x[None] for x in (q, k, v, do)), window, sinks)
    g = torch.Generator(device="cuda").manual_seed(1)
    for n, (x, grad) in enumerate(zip((q, k, v), got[1:])):
        d = torch.randn(x.shape, device="cuda", generator=g, dtype=torch.float64)
        eps = 1e-4
        loss = []
        for sign in (1, -1):
            ins = [q.double(), k.double(), v.double()]
            ins[n] = ins[n] + sign * eps * d
            loss.append((reference(*ins, do, window, sinks)[0] * do.double()).sum())
        want = ((loss[0] - loss[1]) / (2 * eps)).item()
        have = (grad[0].double() * d).sum().item()
        # each gradient element is off by under 2 half steps of its size; along a random direction the
        # errors add up as their norm does, and 8 half steps of it are four of its standard deviations
        assert abs(have - want) < 8 * half_step(torch.float16) * grad.double().norm().item()


def test_strided_views_and_the_mma_kernels():
    from fold_attention_b200.backward import attention_forward, prepare_backward

    S, H, HKV, D, window, sinks = 777, 4, 2, 128, 200, 6
    big = torch.randn(1, S, 2 * (H + 2 * HKV), D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).bfloat16()
    q, k, v = big[:, :, :H], big[:, :, H:H + HKV], big[:, :, H + HKV:H + 2 * HKV]
    do = big[:, :, H + 2 * HKV:2 * H + 2 * HKV]
    want = reference(q[0], k[0], v[0], do[0], window, sinks)
    tr = lambda x: x.transpose(1, 2)  # noqa: E731
    for kernel in ("sm100", "mma"):
        o, lse = attention_forward(q, k, v, causal=True, window=window, sinks=sinks, kernel=kernel)
        run = prepare_backward(tr(q), tr(k), tr(v), tr(o), tr(do), lse, causal=True, window=window, sinks=sinks, kernel=kernel)
        grads = [tr(x) for x in run()]
        run.check()
        check([o[0], *(x[0] for x in grads)], want, torch.bfloat16)
        # the same launch again, and from a graph
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            with torch.cuda.graph(g, stream=side):
                run()
        first = [x.clone() for x in grads]
        for x in grads:
            x.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, grads))


def test_values_under_masks_of_all_sizes_stay_finite():
    """Large scores: a row whose window drops its largest key must not keep its reference."""
    S, D = 512, 128
    q, k, v, do = inputs(S, 1, 1, D, torch.bfloat16, seed=2)
    k[::97] *= 30
    got = run_dense(*(x[None] for x in (q, k, v, do)), 16, 1)
    want = reference(q, k, v, do, 16, 1)
    assert all(torch.isfinite(x).all() for x in got)
    # scores reach a few hundred: an fp32 product of 128 bf16 terms is off by 2^-24 of its terms' size, a
    # weight by that times the score; well inside the 16-bit roundings counted above
    check([x[0] for x in got], want, torch.bfloat16)


@pytest.mark.parametrize("D", [128, 64])
def test_broadcast_heads_and_odd_strides(D):
    """One KV head's tensors expanded over four, queries in a view whose rows sit off the 16-byte boundary."""
    import fold_attention_b200 as fa

    S, window, sinks, dt = 300, 50, 2, torch.bfloat16
    q, k, v, do = inputs(S, 4, 1, D, dt, seed=4)
    wide = torch.zeros(1, S, 4, D + 3, device="cuda", dtype=dt)
    wide[..., 3:] = q[None]
    x = [wide[..., 3:].detach().requires_grad_(), k[None].clone().requires_grad_(), v[None].clone().requires_grad_()]
    out = fa.fold_attn_func(x[0], x[1].expand(1, S, 4, D), x[2].expand(1, S, 4, D), causal=True, window=window, sinks=sinks)
    got = (out.detach(), *torch.autograd.grad(out, x, do[None]))
    # four heads' gradients are added up in 16 bits: three more roundings of a sum, each half a step
    want = reference(q, k, v, do, window, sinks)
    eps = half_step(dt)
    for name, a, b, steps in zip(("out", "dq", "dk", "dv"), got, want, (1, 2, 5, 5)):
        slack = {"dq": want[4], "dk": want[5]}.get(name)
        tol = steps * eps * b.norm().item() + (0 if slack is None else slack.norm().item() * eps)
        assert (a[0].double() - b).norm().item() <= tol, name


def test_on_another_stream_and_captured_beside_an_eager_graph():
    import fold_attention_b200 as fa

    S, window, sinks = 500, 70, 3
    q, k, v, do = (t[None] for t in inputs(S, 4, 2, 128, torch.bfloat16, seed=6))
    want = run_dense(q, k, v, do, window, sinks)
    x = [t.clone().requires_grad_() for t in (q, k, v)]
    eager = fa.fold_attn_func(*x, causal=True, window=window, sinks=sinks)        # lives on while the graph is captured
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = [t.detach().clone().requires_grad_() for t in x]
        other = fa.fold_attn_func(*y, causal=True, window=window, sinks=sinks)
        grads = torch.autograd.grad(other, y, do)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip((other, *grads), want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            z = [t.detach().requires_grad_() for t in x]
            out = fa.fold_attn_func(*z, causal=True, window=window, sinks=sinks)
            captured = torch.autograd.grad(out, z, do)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip((out, *captured), want))
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(eager, x, do), want[1:]))


@pytest.mark.parametrize("D", [128, 64])
def test_rows_behind_the_last_sequence_are_zeros(D):
    import fold_attention_b200 as fa

    lens, window, sinks, pad = [100, 0, 70], 20, 2, 37
    q, k, v, do = inputs(sum(lens) + pad, 4, 2, D, torch.bfloat16, seed=11)
    cu = torch.tensor([0, 100, 100, 170], device="cuda", dtype=torch.int32)
    x = [t.clone().requires_grad_() for t in (q, k, v)]
    torch.full((4 << 20,), float("nan"), device="cuda")        # what the allocator hands out next is not zero
    out = fa.fold_attn_varlen_func(*x, cu, max_seqlen_q=100, causal=True, window=window, sinks=sinks)
    got = (out.detach(), *torch.autograd.grad(out, x, do))
    assert all(not t[170:].any() for t in got)
    for sl in (slice(0, 100), slice(100, 170)):
        check([t[sl] for t in got], reference(q[sl], k[sl], v[sl], do[sl], window, sinks), torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [128, 96])
def test_one_visible_key_has_no_score_gradient(D, dtype):
    """P is 1 whatever the score: dq and dk are zero, not the rounding of two sums that cancel."""
    import fold_attention_b200 as fa

    q, k, v, do = (t[None] for t in inputs(200, 4, 2, D, dtype, seed=3))
    x = [t.clone().requires_grad_() for t in (q, k, v)]
    dq, dk, dv = torch.autograd.grad(fa.fold_attn_func(*x, causal=True, window=1), x, do)
    assert not dq.any() and not dk.any() and dv.any()
    x = [t.clone().requires_grad_() for t in (q[0, :3], k[0, :3], v[0, :3])]
    cu = torch.arange(4, device="cuda", dtype=torch.int32)                     # three sequences of one token
    out = fa.fold_attn_varlen_func(*x, cu, max_seqlen_q=1, causal=True, window=50, sinks=2)
    dq, dk, dv = torch.autograd.grad(out, x, do[0, :3])
    assert not dq.any() and not dk.any() and dv.any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [128, 96, 64])
@pytest.mark.parametrize("lens,window,sinks", [([1000], 2, 0), ([3] * 100, 50, 0), ([300, 5], 3, 1)])
def test_few_visible_keys_keep_their_gradients_precision(lens, window, sinks, D, dtype):
    """Delta comes from the unrounded output: what is left is the rounding of dS and of the results. Each is at most half
    a step, 0.58 of one in the root mean square, so two in a row make 0.82 of the gradient's norm where the terms' signs
    are independent; 0.85 and 2^-15 for the softmax's fp32 are allowed. (O rounded to 16 bits would add 0.7 half steps at two keys a
    query and 2 at sequences of three tokens.)"""
    import fold_attention_b200 as fa

    q, k, v, do = inputs(sum(lens), 4, 2, D, dtype, seed=5)
    x = [t.clone().requires_grad_() for t in (q, k, v)]
    cu = torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), device="cuda", dtype=torch.int32)
    out = fa.fold_attn_varlen_func(*x, cu, max_seqlen_q=max(lens), causal=True, window=window, sinks=sinks)
    got = torch.autograd.grad(out, x, do)
    at, want = 0, []
    for n in lens:
        sl = slice(at, at + n)
        want.append(reference(q[sl], k[sl], v[sl], do[sl], window, sinks))
        at += n
    half = torch.finfo(dtype).eps / 2
    for g, w in zip(got[:2], [torch.cat([r[i] for r in want]) for i in (1, 2)]):
        assert (g.double() - w).norm() <= (0.85 * half + 2 ** -15) * w.norm()


@pytest.mark.parametrize("where", ["tail", "neighbour"])
@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("window,sinks", [(100, 3), (500, 0), (30, 200)])
def test_what_lies_behind_a_sequence_does_not_reach_it(window, sinks, D, where):
    """NaN and infinities in the rows behind a packed sequence, the next one's or nobody's: its results keep their bits."""
    import fold_attention_b200 as fa

    total = 470 + (60 if where == "tail" else 0)
    live = 470 if where == "tail" else 300
    cu = torch.tensor([0, 300, 470], device="cuda", dtype=torch.int32)
    clean = inputs(total, 4, 2, D, torch.bfloat16, seed=4)

    def run(q, k, v, do):
        x = [t.clone().requires_grad_() for t in (q, k, v)]
        out = fa.fold_attn_varlen_func(*x, cu, max_seqlen_q=300, causal=True, window=window, sinks=sinks)
        return (out.detach(), *torch.autograd.grad(out, x, do))

    want = run(*clean)
    for n in range(4):
        for value in (float("nan"), float("inf")):
            bad = [t.clone() for t in clean]
            bad[n][live:] = value
            assert all(torch.equal(a[:live], b[:live]) for a, b in zip(want, run(*bad))), (n, value)


@pytest.mark.parametrize("D", [128, 64])
def test_tensors_off_a_16_byte_boundary(D):
    import fold_attention_b200 as fa

    S, H, HKV, window, sinks = 200, 4, 2, 50, 2
    t = [x[None] for x in inputs(S, H, HKV, D, torch.bfloat16, seed=8)]
    want = run_dense(*t, window, sinks)
    off = []
    for x in t:
        flat = torch.empty(x.numel() + 1, device="cuda", dtype=x.dtype)
        flat[1:] = x.flatten()
        off.append(flat[1:].view(x.shape))
        assert off[-1].data_ptr() % 16
    x = [y.detach().requires_grad_() for y in off[:3]]
    out = fa.fold_attn_func(*x, causal=True, window=window, sinks=sinks)
    got = (out.detach(), *torch.autograd.grad(out, x, off[3]))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
