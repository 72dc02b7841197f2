"""Chunks over the cache where they can go wrong: an 8-bit V's scale, NaN, what a request is batched with."""

import pytest
import torch

pytestmark = pytest.mark.gpu

from test_chunk_gpu import Story, close, cumulative, make  # noqa: E402


@pytest.mark.parametrize("size", [1e-3, 1.0, 3e3])
@pytest.mark.parametrize("D", [64, 128])
def test_pieces_of_a_prompt_set_the_8_bit_scale_that_the_prompt_would(size, D):
    """An empty 8-bit cache without v_scale, filled by chunks. With a power of two above V's largest value a plane's
    rounding is half a step of e4m3 (2^-4 of the value) and the second plane's 2^-4 of that remainder, 2^-8 in all, down to
    values 2^-9 of the scale's unit, of which a normal V this size has few: the norm is within 2^-8."""
    import fold_attention_b200 as fa
    from fold_attention_b200 import decode

    g = torch.Generator(device="cuda").manual_seed(4)
    n = [200, 1, 77]
    k, v = make(n, 2, D, torch.bfloat16, g), make(n, 2, D, torch.bfloat16, g, scale=size)
    a, b = (fa.FoldKVCache(3, 4, 2, D, 300, v8=True, page_size=64) for _ in range(2))
    a.write_prompt(k, v, cumulative(n), n)
    zeros = torch.zeros(1, 2, D, device="cuda", dtype=torch.bfloat16)
    b.append_chunk(zeros, zeros, cumulative([0, 1, 0]), [0, 1, 0])          # zeros say nothing about the scale
    at = [0, 200, 201]
    first = torch.cat([torch.arange(at[0], 200), torch.arange(at[2], 278)]).cuda()
    b.append_chunk(k[first], v[first], cumulative([200, 0, 77]), [200, 0, 77])
    assert b.v_scale == decode.write.v_scale_for(v[first], 2.0)
    assert a.v_scale == decode.write.v_scale_for(v, 2.0)
    slots = (b.page_table[0, torch.arange(200, device="cuda") // 64] * 64 + torch.arange(200, device="cuda") % 64).int()
    _, back = decode.read_tokens(slots, 64, 2, b.ka, b.kb, b.va, b.vb, b.ek, v_scale=b.v_scale, dtype=torch.float32)
    assert (back.double() - v[:200].double()).norm() <= 2.0 ** -8 * v[:200].double().norm()
    kept = b.v_scale                                                           # and later chunks keep it
    b.append_chunk(k[:3], v[:3] * 0.01, cumulative([1, 1, 1]), [1, 1, 1])
    assert b.v_scale == kept


def test_a_captured_first_chunk_of_an_8_bit_cache_is_refused():
    import fold_attention_b200 as fa

    c = fa.FoldKVCache(1, 4, 2, 64, 64, v8=True, page_size=16, pages=4)
    g = torch.Generator(device="cuda").manual_seed(4)
    q, k, v = (make([3], h, 64, torch.bfloat16, g) for h in (4, 2, 2))
    cu, graph, side = cumulative([3]), torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with pytest.raises(ValueError, match="v_scale"):
        with torch.cuda.stream(side):
            with torch.cuda.graph(graph, stream=side):
                c.extend(q, k, v, cu, [3])
    assert c.lens == [0] and c.seq_lens.tolist() == [0] and c.taken.tolist() == [0]
    c.extend(q, k, v, cu, [3])


@pytest.mark.parametrize("D", [64, 128])
def test_a_nan_in_v_stays_one_in_fp16(D):
    import fold_attention_b200 as fa
    from fold_attention_b200 import decode

    dt, g = torch.float16, torch.Generator(device="cuda").manual_seed(4)
    c = fa.FoldKVCache(1, 2, 2, D, 640, page_size=16)
    q, k, v = (make([300], 2, D, dt, g) for _ in range(3))
    v[7] = float("nan")
    out = c.extend(q, k, v, cumulative([300]), [300])              # more than 128 rows: dequantised to fp16
    assert torch.isnan(out[8:]).all()
    assert torch.isnan(c.attend_chunk(q[-2:], cumulative([2]), [2])).all()
    slots = torch.tensor([6, 7], device="cuda", dtype=torch.int32)
    for t in (torch.float16, torch.bfloat16, torch.float32):
        _, back = decode.read_tokens(slots, 16, 2, c.ka, c.kb, c.va, c.vb, c.ek, dtype=t)
        assert torch.isnan(back[1]).all() and torch.isfinite(back[0]).all()
    c.va.fill_(1e30)                                               # beyond fp16: the largest it has
    c.va[0] = -1e30
    _, back = decode.read_tokens(slots - 6, 16, 2, c.ka, c.kb, c.va, c.vb, c.ek, dtype=torch.float16)
    assert (back[1] == 65504).all() and (back[0, 0] == -65504).all()


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("v8", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_query_that_is_no_number_gives_none(value, v8, dtype):
    """In the short chunks' kernel as in the long ones': the row alone, and nothing beside it."""
    import fold_attention_b200 as fa

    g = torch.Generator(device="cuda").manual_seed(4)
    c = fa.FoldKVCache(2, 8, 2, 128, 2000, page_size=64, v8=v8, v_scale=0.25 if v8 else None)
    n = [1500, 200]
    c.append_chunk(*(make(n, 2, 128, dtype, g) for _ in range(2)), cumulative(n), n)
    for rows in ([3, 1], [20, 30], [200, 150]):
        q = make(rows, 8, 128, dtype, g)
        want = c.attend_chunk(q, cumulative(rows), rows)
        bad = q.clone()
        bad[rows[0] - 1, 5, 17] = value
        got = c.attend_chunk(bad, cumulative(rows), rows)
        assert torch.isnan(got[rows[0] - 1, 5]).all()
        got[rows[0] - 1, 5] = want[rows[0] - 1, 5]
        assert torch.equal(got, want), rows


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D", [64, 128])
def test_a_short_request_is_as_right_beside_a_wide_one(D, dtype):
    """Alone it is attended from the codes, beside a wide one or among many its keys may be rounded or cut
    elsewhere: other bits, within the same tolerance."""
    for others in ([], [600], [600, 3, 1], [2] * 40):
        st = Story(1 + len(others), 8, 2, D, 1600, dtype=dtype, page_size=64, v8=True, seed=D)
        st.extend([901] + [max(n, 30) for n in others])
        st.extend([3] + others)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("counts,lens", [([1, 260], [1, 200]), ([3, 9], [3, 4]), ([40, 5], [40, 2])])
def test_counts_that_q_has_no_rows_for_touch_no_row(D, counts, lens):
    """cu_seqlens says more than the host's counts and q's rows: the request is left alone, the others are answered,
    and where the kernel has a status word it is raised."""
    st = Story(2, 8, 2, D, 600, page_size=64, seed=2)
    st.extend([90, 300])
    q, k, v = st.tokens(lens)
    st.c.append_chunk(k, v, cumulative(lens), lens)
    room = torch.zeros(sum(counts) + 8, 8, D, device="cuda", dtype=st.dt)          # (what lies behind q is this test's)
    room[:sum(lens)] = q
    out = st.c.attend_chunk(room[:sum(lens)], cumulative(counts), lens)
    close(out[:lens[0]], st.want(q, lens)[:lens[0]], st.dt)
    if D == 128 or max(lens) <= 32:
        assert st.c._chunk_status.item() == 1
        st.c.check_status = True
        from fold_attention_b200._lib import FoldLibraryError

        with pytest.raises(FoldLibraryError):
            st.c.attend_chunk(room[:sum(lens)], cumulative(counts), lens)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("v8", [False, True])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rows", [1, 200])
@pytest.mark.parametrize("gap", [16.0, 17.6])
def test_many_weights_far_below_one(gap, rows, D, v8, dtype):
    """N keys of logit 0 under one of `gap`: the one's value is 0, the others' 1, so the output is their share w / (1 + w)
    with w = N e^-gap, 0.6 % at 17.6. Each of their weights may lose 2^-32 of the largest to fp16's least step, so N 2^-32 in
    all, beside the roundings of a weight and of the output, half a step each, and fp32's of a sum of N terms in
    128s: 2^-24 (128 + N / 128) of it at most."""
    import math

    import fold_attention_b200 as fa
    from fold_attention_b200 import decode

    N = 1 << 18
    c = fa.FoldKVCache(1, 1, 1, D, N, v8=v8, v_scale=0.25 if v8 else None, page_size=256)
    k = torch.zeros(N, 1, D, device="cuda", dtype=dtype)
    v = torch.ones_like(k)
    v[0], k[0, 0, 0] = 0, 16.0
    c.append_chunk(k, v, cumulative([N]), [N])
    q = torch.zeros(rows, 1, D, device="cuda", dtype=dtype)
    q[:, 0, 0] = gap * math.sqrt(D) / 16.0
    one = torch.zeros(1, device="cuda", dtype=torch.int32)
    key, _ = decode.read_tokens(one, 256, 1, c.ka, c.kb, c.va, c.vb, c.ek, v_scale=c.v_scale, dtype=torch.float32)
    x = (q[0, 0].double() @ key[0, 0].double()).item() / math.sqrt(D)
    # logits of fp32 and codes of 16 bits: 2^-15 of x either way; the wide path rounds the key to 16 bits too
    half = torch.finfo(dtype).eps / 2
    slack = x * (2.0 ** -15 + (half if rows > 128 else 0))
    seen = torch.arange(N - rows, N, device="cuda", dtype=torch.float64)
    share = seen * math.exp(-x) / (1 + seen * math.exp(-x))
    got = c.attend_chunk(q, cumulative([rows]), [rows])[:, 0].double()
    tol = share * (2 * half + 2.0 ** -24 * (128 + N / 128) + math.expm1(slack)) + N * 2.0 ** -32
    assert ((got - share[:, None]).abs() <= tol[:, None]).all(), ((got - share[:, None]).abs().max(1).values / tol).max()
