"""Chunks of new tokens over the paged, quantised cache (`FoldKVCache.extend`), with and without a sliding
window, against 64-bit attention over the values the cache's codes stand for.

Tolerance. Errors are roundings to 16 bits, each at most half a step (2^-8 bf16, 2^-11 fp16) and about 0.42 of one in
the root mean square: of the output, of the weights, of V (an 8-bit V's two planes; exact for a bf16 V) and of K,
which moves a logit by 0.42 half steps of its terms' root sum of squares: about 1 for unit normal q and k, 2 with the few large
keys. An output of independent V is as large as the root sum of squares of its terms, so the four add up in quadrature
to under 0.42 sqrt(1 + 1 + 1 + 4) = 1.1 half steps; 2 are allowed."""

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import cache_format as cf  # noqa: E402

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def dev32(x):
    return torch.tensor(x, device="cuda", dtype=torch.int32)


def cumulative(lens):
    return dev32([0] + list(np.cumsum(lens)))


def make(lens, heads, D, dtype, gen, scale=1.0):
    return (scale * torch.randn(sum(lens), heads, D, device="cuda", generator=gen)).to(dtype)


def values_of(k, v, v8, evs):
    """What the cache's codes of k, v (n, HKV, D) stand for, in 64 bits on the GPU."""
    D = k.shape[-1]
    pa, pb, e = cf.key_planes(k.float().cpu().numpy())
    x = (pa.astype(np.float64) + pb.astype(np.float64) / 256) * e[..., None].astype(np.float64)
    had = np.ones((1, 1))
    while had.shape[0] < D:
        had = np.block([[had, had], [had, -had]])
    kd = torch.from_numpy(x @ had / np.sqrt(D)).cuda()
    if v8:
        a, b = cf.e4m3_planes(v.float().cpu().numpy(), evs)
        vd = torch.from_numpy((cf.e4m3_decode(a).astype(np.float64) + cf.e4m3_decode(b).astype(np.float64) / 8) * evs).cuda()
    else:
        vd = v.to(torch.bfloat16).double()
    return kd, vd


def attend(q, k, v, window, sinks):
    """q (n, H, D) at the last positions of k, v (L, HKV, D), 64 bits."""
    n, H, D = q.shape
    L, HKV = k.shape[:2]
    i = torch.arange(L - n, L, device="cuda")[:, None]
    j = torch.arange(L, device="cuda")[None]
    hide = j > i
    if window:
        hide = hide | ((i - j >= window) & (j >= sinks))
    s = torch.einsum("ihd,jhd->hij", q.double(), k.repeat_interleave(H // HKV, 1)) / math.sqrt(D)
    return torch.einsum("hij,jhd->ihd", torch.softmax(s.masked_fill(hide, -math.inf), -1), v.repeat_interleave(H // HKV, 1))


def close(got, want, dtype, what=""):
    assert torch.isfinite(got).all(), what
    err, size = (got.double() - want).norm().item(), want.norm().item()
    tol = 2 * torch.finfo(dtype).eps / 2
    assert err <= tol * size, (what, err / size, tol)


class Story:
    """A cache and the tokens each request has brought so far."""

    def __init__(self, B, H, HKV, D, max_len, *, v8=False, dtype="bf16", seed=0, garbage=True, **kw):
        import fold_attention_b200 as fa

        self.dt, self.v8, self.evs = DT[dtype], v8, 0.25 if v8 else 1.0
        self.c = fa.FoldKVCache(B, H, HKV, D, max_len, v8=v8, v_scale=self.evs if v8 else None, **kw)
        if "pages" not in kw:
            self.c.page_table.copy_(torch.randperm(self.c.page_table.numel(), device="cuda").int().view_as(self.c.page_table))
        if garbage:     # whatever an earlier owner of the pool left: every bit set (NaN in both of V's types)
            for t in (self.c.ka, self.c.kb, self.c.ek, self.c.va, self.c.vb):
                if t is not None:
                    t.view(torch.uint8).fill_(0xFF)
        self.g = torch.Generator(device="cuda").manual_seed(seed)
        self.H, self.HKV, self.D, self.B = H, HKV, D, B
        self.k = [torch.empty(0, HKV, D, device="cuda", dtype=self.dt) for _ in range(B)]
        self.v = [x.clone() for x in self.k]

    def tokens(self, new):
        q, k, v = (make(new, h, self.D, self.dt, self.g) for h in (self.H, self.HKV, self.HKV))
        k[::53] *= 4
        self.remember(k, v, new)
        return q, k, v

    def remember(self, k, v, new):
        at = 0
        for b, n in enumerate(new):
            self.k[b], self.v[b] = torch.cat((self.k[b], k[at:at + n])), torch.cat((self.v[b], v[at:at + n]))
            at += n

    def want(self, q, new):
        out, at = [], 0
        for b, n in enumerate(new):
            if n:
                out.append(attend(q[at:at + n], *values_of(self.k[b], self.v[b], self.v8, self.evs), self.c.window, self.c.sinks))
            at += n
        return torch.cat(out)

    def extend(self, new):
        import fold_attention_b200 as fa

        q, k, v = self.tokens(new)
        got = fa.fold_attn_with_kvcache(q, self.c, k, v, cu_seqlens=cumulative(new), lens=new)
        assert self.c.lens == [len(x) for x in self.k] and self.c.seq_lens.tolist() == self.c.lens
        close(got, self.want(q, new), self.dt, new)
        return got


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("v8", [False, True])
@pytest.mark.parametrize("D,H,HKV,page", [(128, 8, 2, 64), (64, 6, 2, 16), (128, 4, 4, 128), (128, 16, 1, 192)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (40, 3), (150, 130)])
def test_chunks_of_any_length(dtype, v8, D, H, HKV, page, window, sinks):
    st = Story(4, H, HKV, D, 800, v8=v8, dtype=dtype, page_size=page, window=window, sinks=sinks, seed=D + page)
    st.extend([1, 0, 130, 257])        # an empty cache first, one request without a token
    st.extend([1, 1, 1, 1])
    st.extend([0, 300, 0, 2])
    st.extend([5, 1, 64, 0])
    st.extend([129, 3, 128, 250])


@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (1, 1), (128, 128), (129, 300), (1 << 30, 0)])
@pytest.mark.parametrize("D", [64, 128])
def test_long_contexts(window, sinks, D):
    st = Story(3, 8, 2, D, 5000, v8=True, page_size=256, window=window, sinks=sinks, seed=4)
    old = [4000, 1, 2500]
    q, k, v = st.tokens(old)
    st.c.write_prompt(k, v, cumulative(old), old)
    st.extend([3, 2, 1])
    st.extend([600, 700, 17])
    st.extend([1, 0, 1])


def test_a_chunk_writes_what_a_prompt_writes():
    """The pool after two chunks is the pool after one prompt, to the bit; the V sums to fp32's roundings."""
    import fold_attention_b200 as fa

    B, H, HKV, D = 3, 8, 2, 128
    first, second = [100, 1, 300], [157, 64, 0]
    g = torch.Generator(device="cuda").manual_seed(1)
    both = [a + b for a, b in zip(first, second)]
    k, v = (make(both, HKV, D, torch.bfloat16, g) for _ in range(2))
    cut = lambda x, part: torch.cat([t[:f] if part == 0 else t[f:] for t, f in zip(x.split(both), first)])  # noqa: E731
    caches = []
    for way in range(2):
        c = fa.FoldKVCache(B, H, HKV, D, 400, depth=12.0, tail=None, page_size=64)
        if way:
            c.append_chunk(cut(k, 0), cut(v, 0), cumulative(first))
            c.append_chunk(cut(k, 1), cut(v, 1), cumulative(second), second)
        else:
            c.write_prompt(k, v, cumulative(both), both)
        caches.append(c)
    a, b = caches
    for name in ("ka", "kb", "ek", "va", "seq_lens"):
        assert torch.equal(getattr(a, name), getattr(b, name)), name
    want = torch.stack([t.double().sum(0) for t in v.split(both)]).view(B * HKV, D)
    size = torch.stack([t.double().abs().sum(0) for t in v.split(both)]).view(B * HKV, D)
    # a sum of n terms in any order: at most n - 1 roundings of partial sums no larger than the terms' own sum
    assert ((b.vsum.double() - want).abs() <= 460 * 2.0 ** -24 * size).all()
    n = torch.tensor(both, device="cuda").repeat_interleave(HKV)[:, None]
    assert ((b.vmean.double() - want / n).abs() <= 462 * 2.0 ** -24 * size / n).all()
    # the ordinary decode goes on from there
    q, kn, vn = (make([1] * B, h, D, torch.bfloat16, g) for h in (H, HKV, HKV))
    x, y = a.decode(q, kn, vn), b.decode(q, kn, vn)
    # the same keys and codes; only the mean that dropped mass re-enters at differs, in its last bits
    assert (x.double() - y.double()).norm() <= torch.finfo(torch.bfloat16).eps * x.double().norm()


def test_what_the_pool_holds_past_a_request_moves_no_bit():
    outs = []
    for garbage in (False, True):
        st = Story(2, 8, 2, 128, 900, v8=True, page_size=16, seed=6, garbage=garbage)
        st.c.page_table.copy_(torch.arange(st.c.page_table.numel(), device="cuda").int().view_as(st.c.page_table))
        outs.append([st.extend(n) for n in ([200, 1], [1, 1], [33, 400])])
    for a, b in zip(*outs):
        assert torch.equal(a, b)


def test_a_request_alone_and_in_a_batch():
    """A request's chunk is the same bits whoever it is batched with (and in whatever pages it lies)."""
    st = Story(3, 8, 2, 128, 900, page_size=64, seed=8)
    st.extend([300, 7, 120])
    q, k, v = st.tokens([200, 30, 150])
    got = st.c.extend(q, k, v, cumulative([200, 30, 150]), [200, 30, 150])
    one = Story(1, 8, 2, 128, 900, page_size=64)
    kk, vv = st.k[2], st.v[2]
    one.c.append_chunk(kk, vv, cumulative([270]))
    assert torch.equal(one.c.attend_chunk(q[230:], cumulative([150])), got[230:])


def test_a_shared_pool_hands_out_pages():
    st = Story(3, 4, 2, 64, 640, page_size=32, pages=24, seed=3)
    st.extend([1, 100, 31])
    st.extend([40, 0, 1])
    st.extend([1, 1, 1])
    for _ in range(34):         # across page borders, a token at a time
        q, k, v = st.tokens([1, 1, 1])
        got = st.c.decode(q, k, v)
    close(got, st.want(q, [1, 1, 1]), st.dt)
    pages = sum(-(-n // 32) for n in st.c.lens)
    assert st.c.taken.tolist() == [pages]
    used = [p for b, n in enumerate(st.c.lens) for p in st.c.page_table[b, :-(-n // 32)].tolist()]
    assert sorted(used) == list(range(pages))          # nobody shares a page
    before = list(st.c.lens), st.c.taken.tolist(), st.c.ka.clone()
    with pytest.raises(ValueError, match="pool has 24"):
        st.c.append_chunk(*(make([500, 0, 0], 2, 64, st.dt, st.g) for _ in range(2)), cumulative([500, 0, 0]), [500, 0, 0])
    assert (list(st.c.lens), st.c.taken.tolist()) == before[:2] and torch.equal(st.c.ka, before[2])
    # a new prompt has the whole pool again
    k, v = (make([700], 2, 64, st.dt, st.g) for _ in range(2))
    prompt = [600, 60, 40]
    st.k, st.v = ([x[:0] for x in y] for y in (st.k, st.v))
    st.remember(k, v, prompt)
    st.c.write_prompt(k, v, cumulative(prompt), prompt)
    st.extend([2, 3, 20])


@pytest.mark.parametrize("D,page,v8", [(128, 128, True), (64, 16, False)])
def test_a_windowed_layer_prefills_and_decodes(D, page, v8):
    B, H, HKV, window, sinks = 3, 8, 2, 70, 5
    st = Story(B, H, HKV, D, 600, v8=v8, page_size=page, window=window, sinks=sinks, seed=12)
    prompt = [300, 1, 150]
    q, k, v = st.tokens(prompt)
    got = st.c.prefill(q, k, v, cumulative(prompt))
    want = torch.cat([attend(a, b.double(), c.double(), window, sinks) for a, b, c in zip(q.split(prompt), k.split(prompt), v.split(prompt))])
    close(got, want, st.dt)
    import fold_attention_b200 as fa

    for _ in range(3):
        q, k, v = st.tokens([1] * B)
        got = fa.fold_attn_with_kvcache(q[:, None], st.c, k[:, None], v[:, None])
        assert got.shape == (B, 1, H, D)
        close(got[:, 0], st.want(q, [1] * B), st.dt)
    st.c.append(*st.tokens([1] * B)[1:])
    q = make([1] * B, H, D, st.dt, st.g)
    close(st.c.attend(q), st.want(q, [1] * B), st.dt)


@pytest.mark.parametrize("new", [[1, 1, 1], [9, 0, 40]])
@pytest.mark.parametrize("window", [None, 50])
def test_a_captured_step_replays_on_longer_requests(new, window):
    """The captured call reads and moves the lengths on the device: every replay appends and attends anew."""
    st = Story(3, 8, 2, 128, 700, v8=True, page_size=64, window=window, sinks=2 if window else 0, seed=2)
    st.extend([100, 1, 260])
    sq, sk, sv = (make(new, h, 128, st.dt, st.g) for h in (8, 2, 2))
    cu = cumulative(new)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            out = st.c.extend(sq, sk, sv, cu, new)
    for _ in range(4):
        q, k, v = st.tokens(new)
        for a, b in zip((sq, sk, sv), (q, k, v)):
            a.copy_(b)
        graph.replay()
        close(out, st.want(q, new), st.dt)
    st.c.sync_lens()
    assert st.c.lens == [len(x) for x in st.k]
    st.extend([1, 2, 3])


def test_two_streams_at_once():
    """Two layers' chunks on two streams: workspaces are each call's own."""
    a, b = (Story(2, 8, 2, 128, 1500, page_size=64, seed=s) for s in (1, 2))
    for st in (a, b):
        st.extend([900, 500])
    news = [200, 333]
    ins = [st.tokens(news) for st in (a, b)]
    cu = cumulative(news)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for st, s, (q, k, v) in zip((a, b), streams, ins):
        with torch.cuda.stream(s):
            outs.append(st.c.extend(q, k, v, cu, news))
    torch.cuda.synchronize()
    for st, (q, _, _), out in zip((a, b), ins, outs):
        close(out, st.want(q, news), st.dt)


def test_strided_queries_and_calls_without_lens():
    st = Story(2, 4, 2, 128, 300, page_size=64, seed=7)
    new = [150, 20]
    q, k, v = st.tokens(new)
    wide = torch.zeros(170, 3, 4, 128, device="cuda", dtype=st.dt)
    wide[:, 1] = q
    st.c.append_chunk(k, v, cumulative(new))
    close(st.c.attend_chunk(wide[:, 1], cumulative(new)), st.want(q, new), st.dt)
    # fewer queries than the last chunk brought, and none
    close(st.c.attend_chunk(q[[149, 168, 169]], cumulative([1, 2])), st.want(q[[149, 168, 169]], [1, 2]), st.dt)
    assert st.c.attend_chunk(q[:0], cumulative([0, 0])).shape == (0, 4, 128)
    assert st.c.extend(q[:0], k[:0], v[:0], cumulative([0, 0])).shape == (0, 4, 128)


@pytest.mark.parametrize("v8", [False, True])
def test_hundreds_of_requests(v8):
    """More requests than the short chunks' kernel has threads, most of them without a new token."""
    B = 450
    st = Story(B, 4, 1, 64, 64, v8=v8, page_size=16, seed=5)
    st.extend([b % 5 for b in range(B)])
    st.extend([1 if b % 3 == 0 else 0 for b in range(B)])
    st.extend([40 if b in (7, 440) else b % 2 for b in range(B)])


def test_replays_past_the_end_are_told():
    st = Story(2, 4, 2, 64, 40, page_size=16, pages=6, seed=5)
    st.extend([30, 1])
    q, k, v = (make([1, 1], h, 64, st.dt, st.g) for h in (4, 2, 2))
    cu, graph, side = cumulative([1, 1]), torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            st.c.extend(q, k, v, cu, [1, 1])
    for _ in range(9):
        graph.replay()
    st.c.sync_lens()
    assert st.c.lens == [39, 10]
    for _ in range(9):
        graph.replay()
    with pytest.raises(ValueError, match="max_len=40"):
        st.c.sync_lens()


def test_small_pages_and_one_key():
    """A request of one key, alone: one visible key, whose value is the output to its rounding."""
    st = Story(1, 8, 8, 128, 16, page_size=16, seed=1)
    q, k, v = st.tokens([1])
    got = st.c.extend(q, k, v, cumulative([1]), [1])
    assert torch.equal(got, v)
