"""What the attention operators for long contexts are measured on.

Four operators that a model with long contexts trains and serves through:

* `window`: causal self-attention under a sliding window with a few first tokens that stay
  visible, forward and gradients, dense and packed (`fold_attn_func`, `fold_attn_varlen_func`);
* `chunk`: attention of each request's newest tokens, one or thousands, over the paged, quantised
  cache that already holds them (`FoldKVCache.attend_chunk`), with or without the window;
* `tables`: block tables and the new tokens' slots from request lengths
  (`decode.build_tables`);
* `tokens`: new tokens quantised into the pool at their slots, and read back
  (`decode.write_tokens`, `decode.read_tokens`).

Each case is a dict of plain values. `prepare` makes its inputs, `run` is one pass (in the plain
form, or through the package where `own` is true), `work` counts what a pass cannot do without,
and `exact` gives the outputs in 64 bits.
"""

import math
import random

import numpy as np
import torch

own = False

DEVICE = "cuda"
LOG2E = 1.4426950408889634


# ---- the cases -------------------------------------------------------------------

def listed():
    return [
        # -- sliding window, training
        # a small model's step: launches are what costs
        dict(name="window-small-d64", op="window", batch=2, seq=512, heads=8, kv_heads=8, dim=64, dtype="bf16",
             packed=False, window=128, sinks=4, lens_seed=0),
        # odd everything, the warp-level kernels, three heads a group
        dict(name="window-odd-d96-fp16", op="window", batch=3, seq=1037, heads=6, kv_heads=2, dim=96, dtype="fp16",
             packed=False, window=77, sinks=5, lens_seed=0),
        # packed documents of a training batch, no sinks
        dict(name="window-packed-16k", op="window", batch=6, seq=16384, heads=32, kv_heads=8, dim=128, dtype="bf16",
             packed=True, window=512, sinks=0, lens_seed=3),
        # long sequences, the shape the training path's headline uses
        dict(name="window-8k-sinks", op="window", batch=2, seq=8192, heads=32, kv_heads=8, dim=128, dtype="bf16",
             packed=False, window=1024, sinks=4, lens_seed=0),
        # -- chunks over the cache, serving
        # one token a request under a window: the decode step of a sliding-window layer
        dict(name="chunk-decode-window", op="chunk", batch=64, ctx_lo=1024, ctx_hi=32768, new_lo=1, new_hi=1, heads=32,
             kv_heads=8, dim=128, dtype="bf16", v8=True, page=128, window=1024, sinks=4, lens_seed=5),
        # a few drafted tokens a request, verified in one pass
        dict(name="chunk-verify", op="chunk", batch=32, ctx_lo=1024, ctx_hi=32768, new_lo=3, new_hi=8, heads=32, kv_heads=8,
             dim=128, dtype="bf16", v8=False, page=64, window=0, sinks=0, lens_seed=7),
        # two prompts prefilled piece by piece, late pieces
        dict(name="chunk-prefill-2k", op="chunk", batch=2, ctx_lo=16384, ctx_hi=24576, new_lo=2048, new_hi=2048, heads=32,
             kv_heads=8, dim=128, dtype="bf16", v8=True, page=256, window=0, sinks=0, lens_seed=11),
        # short contexts of a small model, ragged pieces and requests that bring nothing
        dict(name="chunk-ragged-d64-fp16", op="chunk", batch=9, ctx_lo=1, ctx_hi=1500, new_lo=0, new_hi=300, heads=6, kv_heads=2,
             dim=64, dtype="fp16", v8=True, page=16, window=0, sinks=0, lens_seed=13),
        # -- block tables and slots
        # a decode step of a large batch: one token a request
        dict(name="tables-decode", op="tables", batch=256, ctx_lo=1024, ctx_hi=32768, new_lo=1, new_hi=1, page=64, lens_seed=17),
        # a prefill: whole prompts
        dict(name="tables-prefill", op="tables", batch=48, ctx_lo=0, ctx_hi=100, new_lo=1, new_hi=4096, page=16, lens_seed=19),
        # -- tokens into the pool
        dict(name="tokens-decode-v8", op="tokens", tokens=256, kv_heads=8, dim=128, dtype="bf16", v8=True, page=128),
        dict(name="tokens-prefill", op="tokens", tokens=16384, kv_heads=8, dim=128, dtype="bf16", v8=False, page=64),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["window", "window", "chunk", "chunk", "tables", "tokens"])
    if op == "window":
        dim = rng.choice([64, 96, 128, 128])
        kv = rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 2, 3, 4])
        packed = rng.random() < 0.5
        seq = _log_int(rng, 1, 8192)
        batch = rng.randint(1, 2) if not packed else rng.randint(1, 8)
        batch = min(batch, seq)
        return dict(op=op, batch=batch, seq=seq, heads=heads, kv_heads=kv, dim=dim, dtype=rng.choice(["bf16", "fp16"]),
                    packed=packed, window=_log_int(rng, 1, 1024), sinks=rng.choice([0, 1, 4, rng.randint(0, 300)]),
                    lens_seed=rng.randrange(1 << 30))
    if op == "chunk":
        dim = rng.choice([64, 128, 128])
        kv = rng.choice([1, 2, 8])
        heads = kv * rng.choice([1, 3, 4, 8])
        batch = _log_int(rng, 1, 24)
        new_hi = rng.choice([1, rng.randint(1, 16), _log_int(rng, 1, 1024)])
        new_lo = rng.choice([0, 1, new_hi])
        ctx_hi = _log_int(rng, 1, 16384)
        windowed = rng.random() < 0.5
        return dict(op=op, batch=batch, ctx_lo=rng.choice([0, ctx_hi // 2, ctx_hi]), ctx_hi=ctx_hi, new_lo=new_lo, new_hi=new_hi, heads=heads,
                    kv_heads=kv, dim=dim, dtype=rng.choice(["bf16", "fp16"]), v8=rng.random() < 0.5,
                    page=rng.choice([16, 32, 64, 128, 256, 192]), window=_log_int(rng, 1, 2048) if windowed else 0,
                    sinks=rng.choice([0, 4, rng.randint(0, 200)]) if windowed else 0, lens_seed=rng.randrange(1 << 30))
    if op == "tables":
        new_hi = rng.choice([1, _log_int(rng, 1, 1024)])
        return dict(op=op, batch=_log_int(rng, 1, 300), ctx_lo=0, ctx_hi=_log_int(rng, 1, 32768),
                    new_lo=rng.choice([0, 1]), new_hi=new_hi, page=rng.choice([16, 32, 64, 128, 256]), lens_seed=rng.randrange(1 << 30))
    return dict(op=op, tokens=_log_int(rng, 1, 16384), kv_heads=rng.choice([1, 2, 3, 8]), dim=rng.choice([64, 128]),
                dtype=rng.choice(["bf16", "fp16"]), v8=rng.random() < 0.5, page=rng.choice([16, 32, 64, 128, 256]))


def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float16


def _lengths(case):
    """The case's own lengths: packed sequences, or (context before, new tokens) of each request."""
    rng = random.Random(case["lens_seed"])
    if case["op"] == "window":
        if not case["packed"]:
            return [case["seq"]] * case["batch"]
        cuts = sorted(rng.sample(range(1, case["seq"]), case["batch"] - 1))
        return [b - a for a, b in zip([0] + cuts, cuts + [case["seq"]])]
    old = [rng.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["batch"])]
    new = [rng.randint(case["new_lo"], case["new_hi"]) for _ in range(case["batch"])]
    if sum(new) == 0:
        new[0] = 1
    if case["op"] == "chunk":   # a cache that was ever filled holds a token of every request
        old = [max(o, 1) if n == 0 else o for o, n in zip(old, new)]
    return old, new


def _cumulative(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _visible(pos, n_sinks, window):
    """How many keys the token at `pos` sees."""
    if window <= 0 or window > pos:
        return pos + 1
    first = pos - window + 1
    return window + min(n_sinks, first)


def work(case):
    op = case["op"]
    if op == "window":
        pairs = sum(_visible(i, case["sinks"], case["window"]) for n in _lengths(case) for i in range(n))
        rows = sum(_lengths(case))
        size = 2 * case["dim"] * rows * 4 * (case["heads"] + case["kv_heads"])
        return {"bytes": size, "flops": 14 * pairs * case["heads"] * case["dim"]}
    if op == "chunk":
        old, new = _lengths(case)
        keys = pairs = 0
        for o, n in zip(old, new):
            if n == 0:
                continue
            pairs += sum(_visible(o + i, case["sinks"], case["window"]) for i in range(n))
            first = 0 if case["window"] <= 0 else max(0, o - case["window"] + 1)
            keys += o + n - first + min(case["sinks"], first)
        d = case["dim"]
        size = keys * case["kv_heads"] * (4 * d + 2) + 2 * 2 * sum(new) * case["heads"] * d
        return {"bytes": size, "flops": 4 * pairs * case["heads"] * d}
    if op == "tables":
        old, new = _lengths(case)
        p = case["page"]
        grown = sum(-(-(o + n) // p) - -(-o // p) for o, n in zip(old, new))
        touched = sum(-(-(o + n) // p) - o // p for o, n in zip(old, new) if n)
        return {"bytes": 4 * (3 * case["batch"] + 2 * grown + touched + sum(new)), "flops": 4 * sum(new)}
    rows, d = case["tokens"] * case["kv_heads"], case["dim"]
    # k and v in, codes and scales out; codes and scales in, 32-bit values out
    size = rows * (4 * d + (4 * d + 2) + (4 * d + 2) + 8 * d) + 8 * case["tokens"]
    return {"bytes": size, "flops": 2 * rows * d * int(math.log2(d))}


# ---- inputs ----------------------------------------------------------------------

class State:
    pass


def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _randn(gen, *shape, dtype):
    return torch.randn(*shape, generator=gen, device=DEVICE, dtype=torch.float32).to(dtype)


def _keys(gen, n, heads, dim, dtype):
    """Keys of which one in a hundred is large: attention that peaks somewhere."""
    k = torch.randn(n, heads, dim, generator=gen, device=DEVICE)
    big = torch.rand(n, 1, 1, generator=gen, device=DEVICE) < 0.01
    return torch.where(big, 4.0 * k, k).to(dtype)


def _values(gen, n, heads, dim, dtype):
    v = torch.randn(n, heads, dim, generator=gen, device=DEVICE)
    out = torch.rand(n, heads, dim, generator=gen, device=DEVICE) < 0.001
    return torch.where(out, 20.0 * v, v).to(dtype)


V_SCALE = 0.5   # the 8-bit values' power of two: the largest of them stay under 448 of it


def prepare(case, seed):
    st = State()
    st.case = case
    gen = _generator(seed)
    op = case["op"]
    if op == "window":
        _prepare_window(st, case, gen)
    elif op == "chunk":
        _prepare_chunk(st, case, gen, seed)
    elif op == "tables":
        _prepare_tables(st, case, seed)
    else:
        _prepare_tokens(st, case, gen, seed)
    return st


def _prepare_window(st, case, gen):
    dt, d = _dtype(case), case["dim"]
    lens = _lengths(case)
    lead = (sum(lens),) if case["packed"] else (case["batch"], case["seq"])
    st.q = _randn(gen, *lead, case["heads"], d, dtype=dt)
    st.k = _randn(gen, *lead, case["kv_heads"], d, dtype=dt)
    st.v = _randn(gen, *lead, case["kv_heads"], d, dtype=dt)
    st.dout = _randn(gen, *lead, case["heads"], d, dtype=dt)
    st.lens = lens
    st.cu = torch.tensor(_cumulative(lens), device=DEVICE, dtype=torch.int32)


def _prepare_chunk(st, case, gen, seed):
    dt, d, hkv, page = _dtype(case), case["dim"], case["kv_heads"], case["page"]
    old, new = _lengths(case)
    ctx = [o + n for o, n in zip(old, new)]
    per = -(-max(ctx) // page)
    pages = case["batch"] * per
    perm = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    st.table = perm.view(case["batch"], per).to(DEVICE)
    st.old, st.new, st.ctx = old, new, ctx
    st.cu = torch.tensor(_cumulative(new), device=DEVICE, dtype=torch.int32)
    st.q = _randn(gen, sum(new), case["heads"], d, dtype=dt)
    if own:
        from fold_attention_b200 import FoldKVCache

        st.cache = FoldKVCache(case["batch"], case["heads"], hkv, d, per * page, v8=case["v8"], page_size=page,
                               v_scale=V_SCALE if case["v8"] else None, window=case["window"] or None, sinks=case["sinks"])
        st.cache.page_table.copy_(st.table)
        cu = torch.tensor(_cumulative(ctx), device=DEVICE, dtype=torch.int32)
        k = torch.empty(sum(ctx), hkv, d, device=DEVICE, dtype=dt)
        v = torch.empty_like(k)
    else:
        st.ka = torch.zeros(pages, page, hkv, d, device=DEVICE, dtype=torch.int8)
        st.kb = torch.zeros_like(st.ka)
        st.ek = torch.zeros(pages, page, hkv, device=DEVICE)
        vt = torch.float8_e4m3fn if case["v8"] else torch.bfloat16
        st.va = torch.zeros(pages, page, hkv, d, device=DEVICE).to(vt)
        st.vb = torch.zeros(pages, page, hkv, d, device=DEVICE).to(vt) if case["v8"] else None
    at = 0
    for b, n in enumerate(ctx):
        kk, vv = _keys(gen, n, hkv, d, dt), _values(gen, n, hkv, d, dt)
        if own:
            k[at:at + n], v[at:at + n] = kk, vv
        else:
            pos = torch.arange(n, device=DEVICE)
            pg, sl = st.table[b, pos // page].long(), pos % page
            a, c, e = _key_codes(kk)
            st.ka[pg, sl], st.kb[pg, sl], st.ek[pg, sl] = a.to(torch.int8), c.to(torch.int8), e
            if case["v8"]:
                x, y = _value_codes(vv)
                st.va.view(torch.uint8)[pg, sl] = x.view(torch.uint8)
                st.vb.view(torch.uint8)[pg, sl] = y.view(torch.uint8)
            else:
                st.va[pg, sl] = vv.to(torch.bfloat16)
        at += n
    if own:
        st.cache.write_prompt(k, v, cu, ctx)


def _prepare_tables(st, case, seed):
    old, new = _lengths(case)
    page = case["page"]
    ctx = [o + n for o, n in zip(old, new)]
    per = -(-max(ctx) // page)
    total = sum(-(-c // page) for c in ctx) + 7
    rng = np.random.default_rng(seed)
    free = rng.permutation(total).astype(np.int32)
    table = np.zeros((case["batch"], per), np.int32)
    taken = 0
    for b, o in enumerate(old):   # what earlier steps handed out
        n = -(-o // page)
        table[b, :n] = free[taken:taken + n]
        taken += n
    st.table = torch.from_numpy(table).to(DEVICE)
    st.free = torch.from_numpy(free).to(DEVICE)
    st.taken = torch.tensor([taken], device=DEVICE, dtype=torch.int32)
    st.lens = torch.tensor(old, device=DEVICE, dtype=torch.int32)
    st.cu = torch.tensor(_cumulative(new), device=DEVICE, dtype=torch.int32)
    st.total = sum(new)


def _prepare_tokens(st, case, gen, seed):
    dt, d, hkv, page, n = _dtype(case), case["dim"], case["kv_heads"], case["page"], case["tokens"]
    pages = -(-n // page) + 1
    st.k, st.v = _keys(gen, n, hkv, d, dt), _values(gen, n, hkv, d, dt)
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(seed))[:n]
    # pages in any order, a page's tokens in a row
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed + 1))
    t = torch.arange(n)
    slots = order[t // page] * page + t % page if n > page else slots
    st.slots = slots.to(device=DEVICE, dtype=torch.int32)
    rows = pages * page * hkv
    st.ka = torch.zeros(rows, d, device=DEVICE, dtype=torch.int8)
    st.kb = torch.zeros_like(st.ka)
    st.ek = torch.zeros(rows, device=DEVICE, dtype=torch.bfloat16)
    vt = torch.float8_e4m3fn if case["v8"] else torch.bfloat16
    st.va = torch.zeros(rows, d, device=DEVICE).to(vt)
    st.vb = torch.zeros(rows, d, device=DEVICE).to(vt) if case["v8"] else None


# ---- the cache's format, in its own 32-bit steps -----------------------------------

def _rotate(x):
    """The orthonormal Hadamard transform of the last axis, stage by stage."""
    d = x.shape[-1]
    h = 1
    while h < d:
        y = x.view(*x.shape[:-1], d // (2 * h), 2, h)
        x = torch.stack((y[..., 0, :] + y[..., 1, :], y[..., 0, :] - y[..., 1, :]), dim=-2).view(*x.shape[:-1], d)
        h *= 2
    return x * torch.tensor(0.125 if d == 64 else 0.08838834764831845, device=x.device, dtype=x.dtype)


def _key_codes(k):
    """A key's two planes (whole numbers, as floats) and its scale: k rotated = e (a + b / 256)."""
    x = _rotate(k.float())
    e = x.abs().amax(-1).clamp_min(1e-30) * torch.tensor(1.0 / 127.0, device=x.device, dtype=torch.float32)
    bits = ((e.view(torch.int32) + 0xFFFF) >> 16) << 16        # to bf16, upward
    e = bits.view(torch.float32)[..., None]
    a = torch.round((x * (1.0 / e)).clamp(-128.0, 127.0))
    b = torch.round(((x - a * e) * (256.0 / e)).clamp(-128.0, 127.0))
    return a, b, e[..., 0]


def _value_codes(v):
    s = v.float() * (1.0 / V_SCALE)
    a = s.clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    b = ((s - a.float()) * 8.0).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return a, b


# ---- the plain forms ---------------------------------------------------------------

def run(st):
    return {"window": _run_window, "chunk": _run_chunk, "tables": _run_tables, "tokens": _run_tokens}[st.case["op"]](st)


def _run_window(st):
    case = st.case
    if own:
        import fold_attention_b200 as fa

        q, k, v = (x.detach().requires_grad_() for x in (st.q, st.k, st.v))
        if case["packed"]:
            out = fa.fold_attn_varlen_func(q, k, v, st.cu, max_seqlen_q=max(st.lens), causal=True, window=case["window"],
                                           sinks=case["sinks"])
        else:
            out = fa.fold_attn_func(q, k, v, causal=True, window=case["window"], sinks=case["sinks"])
        return (out.detach(), *torch.autograd.grad(out, (q, k, v), st.dout))
    shape_q, shape_k = st.q.shape, st.k.shape
    flat = lambda x: x.reshape(-1, *x.shape[-2:])  # noqa: E731
    outs = [[], [], [], []]
    at = 0
    for n in st.lens:
        part = [flat(x)[at:at + n] for x in (st.q, st.k, st.v, st.dout)]
        for keep, x in zip(outs, _window_plain(*part, case["window"], case["sinks"])):
            keep.append(x)
        at += n
    out, dq, dk, dv = (torch.cat(x) for x in outs)
    return out.view(shape_q), dq.view(shape_q), dk.view(shape_k), dv.view(shape_k)


def _window_plain(q, k, v, dout, window, sinks, block=1024):
    """One sequence, a block of queries at a time against the keys that its window and the sinks hold."""
    n, heads, d = q.shape
    hkv = k.shape[1]
    g, scale, dt = heads // hkv, 1.0 / math.sqrt(d), q.dtype
    qf = q.float().view(n, hkv, g, d).permute(1, 2, 0, 3)          # (hkv, g, n, d)
    df = dout.float().view(n, hkv, g, d).permute(1, 2, 0, 3)
    kf, vf = k.float().transpose(0, 1), v.float().transpose(0, 1)  # (hkv, n, d)
    out, dq = torch.empty_like(qf), torch.empty_like(qf)
    dk, dv = torch.zeros_like(kf), torch.zeros_like(vf)
    pos = torch.arange(n, device=q.device)
    for i0 in range(0, n, block):
        i1 = min(n, i0 + block)
        lo = max(0, i0 - window + 1)
        cols = torch.cat((pos[:min(sinks, lo)], pos[lo:i1]))
        rows = pos[i0:i1, None]
        seen = (cols <= rows) & ((cols > rows - window) | (cols < sinks))
        kb, vb = kf[:, cols], vf[:, cols]                           # (hkv, m, d)
        qb, db = qf[:, :, i0:i1].reshape(hkv, -1, d), df[:, :, i0:i1].reshape(hkv, -1, d)
        s = (qb @ kb.transpose(1, 2)).view(hkv, g, i1 - i0, -1) * scale
        s = torch.where(seen, s, -math.inf)
        p = torch.exp(s - s.amax(-1, keepdim=True))
        p = (p / p.sum(-1, keepdim=True)).view(hkv, -1, cols.numel())
        ob = p @ vb
        dv.index_add_(1, cols, p.transpose(1, 2) @ db)
        ds = p * (db @ vb.transpose(1, 2) - (ob * db).sum(-1, keepdim=True)) * scale
        dk.index_add_(1, cols, ds.transpose(1, 2) @ qb)
        out[:, :, i0:i1] = ob.view(hkv, g, -1, d)
        dq[:, :, i0:i1] = (ds @ kb).view(hkv, g, -1, d)
    back = lambda x: x.permute(2, 0, 1, 3).reshape(n, heads, d).to(dt)  # noqa: E731
    return back(out), back(dq), dk.transpose(0, 1).to(dt), dv.transpose(0, 1).to(dt)


def _run_chunk(st):
    case = st.case
    if own:
        return st.cache.attend_chunk(st.q, st.cu, lens=st.new)
    page, window, sinks = case["page"], case["window"], case["sinks"]
    d, hkv = case["dim"], case["kv_heads"]
    g = case["heads"] // hkv
    out = torch.empty_like(st.q)
    at = 0
    for b, (o, n) in enumerate(zip(st.old, st.new)):
        if n == 0:
            continue
        first = 0 if window <= 0 else max(0, o - window + 1)
        cols = torch.arange(first, o + n, device=DEVICE)
        if first and sinks:
            cols = torch.cat((torch.arange(min(sinks, first), device=DEVICE), cols))
        pg, sl = st.table[b, cols // page].long(), cols % page
        k = ((st.ka[pg, sl].float() + st.kb[pg, sl].float() / 256.0) * st.ek[pg, sl][..., None]).transpose(0, 1)
        if st.vb is not None:
            x, y = (plane.view(torch.uint8)[pg, sl].view(torch.float8_e4m3fn).float() for plane in (st.va, st.vb))
            v = ((x + y / 8.0) * V_SCALE).transpose(0, 1)
        else:
            v = st.va[pg, sl].float().transpose(0, 1)
        for i0 in range(0, n, 512):
            i1 = min(n, i0 + 512)
            q = _rotate(st.q[at + i0:at + i1].float()).view(i1 - i0, hkv, g, d).permute(1, 2, 0, 3).reshape(hkv, -1, d)
            rows = torch.arange(o + i0, o + i1, device=DEVICE)[:, None]
            seen = cols <= rows
            if window > 0:
                seen &= (cols > rows - window) | (cols < sinks)
            s = (q @ k.transpose(1, 2)).view(hkv, g, i1 - i0, -1) / math.sqrt(d)
            s = torch.where(seen, s, -math.inf)
            p = torch.exp(s - s.amax(-1, keepdim=True))
            x = (p.view(hkv, -1, cols.numel()) @ v).view(hkv, g, i1 - i0, d) / p.sum(-1, keepdim=True)
            out[at + i0:at + i1] = x.permute(2, 0, 1, 3).reshape(i1 - i0, hkv * g, d).to(out.dtype)
        at += n
    return out


def _run_tables(st):
    page = st.case["page"]
    if own:
        from fold_attention_b200 import decode

        slots, lens, taken = decode.build_tables(st.cu, st.lens, st.table, page, st.total, free_pages=st.free, taken=st.taken)
        return st.table, slots, lens, taken
    new = st.cu[1:] - st.cu[:-1]
    lens = st.lens + new
    p0, p1 = (st.lens + page - 1) // page, (lens + page - 1) // page
    grown = p1 - p0
    first = torch.cumsum(grown, 0) - grown + st.taken
    col = torch.arange(st.table.shape[1], device=DEVICE)[None, :]
    fresh = (col >= p0[:, None]) & (col < p1[:, None])
    src = (first[:, None] + col - p0[:, None]).clamp(0, st.free.numel() - 1)
    st.table.copy_(torch.where(fresh, st.free[src], st.table))
    t = torch.arange(st.total, device=DEVICE, dtype=torch.int32)
    req = (t[:, None] >= st.cu[None, 1:]).sum(1)
    pos = st.lens[req] + t - st.cu[req]
    slots = st.table[req, pos // page] * page + pos % page
    return st.table, slots.to(torch.int32), lens.to(torch.int32), (st.taken + grown.sum()).to(torch.int32)


def _run_tokens(st):
    page, hkv = st.case["page"], st.case["kv_heads"]
    if own:
        from fold_attention_b200 import decode

        decode.write_tokens(st.k, st.v, st.slots, page, st.ka, st.kb, st.va, st.vb, st.ek, v_scale=V_SCALE if st.vb is not None else 1.0)
        return decode.read_tokens(st.slots, page, hkv, st.ka, st.kb, st.va, st.vb, st.ek,
                                  v_scale=V_SCALE if st.vb is not None else 1.0, dtype=torch.float32)
    slots = st.slots.long()
    head = torch.arange(hkv, device=DEVICE)
    row = ((slots // page)[:, None] * hkv + head) * page + (slots % page)[:, None]
    a, b, e = _key_codes(st.k)
    st.ka[row], st.kb[row], st.ek[row] = a.to(torch.int8), b.to(torch.int8), e.to(torch.bfloat16)
    if st.vb is not None:
        x, y = _value_codes(st.v)
        st.va.view(torch.uint8)[row] = x.view(torch.uint8)
        st.vb.view(torch.uint8)[row] = y.view(torch.uint8)
        v = (st.va.view(torch.uint8)[row].view(torch.float8_e4m3fn).float()
             + st.vb.view(torch.uint8)[row].view(torch.float8_e4m3fn).float() / 8.0) * V_SCALE
    else:
        st.va[row] = st.v.to(torch.bfloat16)
        v = st.va[row].float()
    k = _rotate((st.ka[row].float() + st.kb[row].float() / 256.0) * st.ek[row].float()[..., None])
    return k, v


# ---- in 64 bits --------------------------------------------------------------------

def exact(case, seed):
    op = case["op"]
    st = State()
    st.case = case
    gen = _generator(seed)
    if op == "tables":
        _prepare_tables(st, case, seed)
        return _exact_tables(st)
    if op == "window":
        _prepare_window(st, case, gen)
        return _exact_window(st)
    if op == "chunk":
        return _exact_chunk(case, seed)
    _prepare_tokens(st, case, gen, seed)
    return _key_value(st.k), _value_value(st.v, case["v8"])


def _exact_tables(st):
    """The pages handed out one request and one page at a time."""
    page = st.case["page"]
    old, new = _lengths(st.case)
    table, free = st.table.cpu().tolist(), st.free.cpu().tolist()
    taken, slots = int(st.taken), []
    for b, (o, n) in enumerate(zip(old, new)):
        for at in range(o, o + n):
            if at % page == 0:
                table[b][at // page] = free[taken]
                taken += 1
            slots.append(table[b][at // page] * page + at % page)
    whole = lambda x: torch.tensor(x, dtype=torch.int32, device=DEVICE)  # noqa: E731
    return whole(table), whole(slots), whole([o + n for o, n in zip(old, new)]), whole([taken])


def _exact_window(st):
    """Every pair's score, masked, with 64-bit autograd for the gradients, a head at a time."""
    case = st.case
    g, d = case["heads"] // case["kv_heads"], case["dim"]
    q, k, v, do = (x.reshape(-1, *x.shape[-2:]).double() for x in (st.q, st.k, st.v, st.dout))
    res = [torch.zeros_like(x) for x in (q, q, k, v)]
    at = 0
    for n in st.lens:
        i = torch.arange(n, device=q.device)
        gap = i[:, None] - i[None, :]
        hide = (gap < 0) | ((gap >= case["window"]) & (i[None, :] >= case["sinks"]))
        sl = slice(at, at + n)
        for h in range(case["heads"]):
            a, b, c = (x.clone().requires_grad_() for x in (q[sl, h], k[sl, h // g], v[sl, h // g]))
            w = torch.softmax((a @ b.T).div(math.sqrt(d)).masked_fill(hide, -math.inf), dim=1)
            o = w @ c
            ga, gb, gc = torch.autograd.grad(o, (a, b, c), do[sl, h])
            res[0][sl, h], res[1][sl, h] = o.detach(), ga
            res[2][sl, h // g] += gb
            res[3][sl, h // g] += gc
            del w, o
        at += n
    return tuple(x.view(y.shape) for x, y in zip(res, (st.q, st.q, st.k, st.v)))


def _hadamard(d):
    m = torch.ones(1, 1, dtype=torch.float64)
    while m.shape[0] < d:
        m = torch.cat((torch.cat((m, m), 1), torch.cat((m, -m), 1)))
    return (m / math.sqrt(d)).to(DEVICE)


def _key_value(k):
    """What a key's codes stand for, in the key's own basis: the codes by the format's 32-bit steps, the rest in 64."""
    d = k.shape[-1]
    f = lambda c: torch.tensor(c, dtype=torch.float32, device=k.device)  # noqa: E731
    x = k.float()
    idx = torch.arange(d, device=k.device)
    step = 1
    while step < d:
        other = x.index_select(-1, idx ^ step)
        x = torch.where((idx & step) == 0, x + other, other - x)
        step *= 2
    x = x * f(0.125 if d == 64 else 0.08838834764831845)
    e = torch.maximum(x.abs().max(-1, keepdim=True).values, f(1e-30)) * f(1.0 / 127.0)
    low = e.view(torch.int32) & 0xFFFF
    e = torch.where(low == 0, e, ((e.view(torch.int32) - low) + 0x10000).view(torch.float32))   # to bf16, upward
    a = torch.round(torch.minimum(torch.maximum(x * torch.div(f(1.0), e), f(-128.0)), f(127.0)))
    b = torch.round(torch.minimum(torch.maximum((x - a * e) * torch.div(f(256.0), e), f(-128.0)), f(127.0)))
    return (e.double() * (a.double() + b.double() / 256.0)) @ _hadamard(d)


def _to_e4m3(x):
    """The nearest e4m3 value, ties to the even code."""
    x = x.double().clamp(-448.0, 448.0)
    ulp = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(x / ulp) * ulp


def _value_value(v, v8):
    if not v8:
        return v.to(torch.bfloat16).double()
    s = v.float() / V_SCALE
    a = _to_e4m3(s)
    b = _to_e4m3((s - a.float()) * 8)
    return (a + b / 8.0) * V_SCALE


def _exact_chunk(case, seed):
    """Each request's own keys and values (made again from the seed), dequantised and attended in 64 bits."""
    old, new = _lengths(case)
    d, hkv, dt = case["dim"], case["kv_heads"], _dtype(case)
    g = case["heads"] // hkv
    gen = _generator(seed)
    q = _randn(gen, sum(new), case["heads"], d, dtype=dt).double()
    out = torch.zeros_like(q)
    at = 0
    for o, n in zip(old, new):
        k, v = _keys(gen, o + n, hkv, d, dt), _values(gen, o + n, hkv, d, dt)
        if n == 0:
            continue
        i = torch.arange(o, o + n, device=DEVICE)[:, None]
        j = torch.arange(o + n, device=DEVICE)
        if case["window"] > 0:
            j = j[(j > o - case["window"]) | (j < case["sinks"])]
        k, v, j = _key_value(k[j]), _value_value(v[j], case["v8"]), j[None, :]
        hide = j > i
        if case["window"] > 0:
            hide = hide | ((i - j >= case["window"]) & (j >= case["sinks"]))
        for h in range(case["heads"]):
            w = torch.softmax((q[at:at + n, h] @ k[:, h // g].T / math.sqrt(d)).masked_fill(hide, -math.inf), dim=1)
            out[at:at + n, h] = w @ v[:, h // g]
        at += n
    return out
