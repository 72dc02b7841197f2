"""Block tables and slots built on the device, and tokens written into the pool at their slots and read
back: whole numbers equal a plain implementation's, planes equal the oracle's to the bit, and what is read
back is the codes' value to fp32's roundings (7 adds and one multiply of the rotation, each half a step of
its result, whose size is at most the row's norm: under 8 half steps of 2^-24 of that)."""

import random

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import cache_format as cf  # noqa: E402


def dev32(x):
    return torch.tensor(x, device="cuda", dtype=torch.int32)


def plain_tables(cu, old, table, page, total, free=None, taken=0):
    table = [list(r) for r in table]
    slots = [-1] * total
    for b, o in enumerate(old):
        n = cu[b + 1] - cu[b]
        if free is not None:
            for j in range(-(-o // page), -(-(o + n) // page)):
                if j < len(table[b]) and taken < len(free):
                    table[b][j] = free[taken]
                elif j < len(table[b]):
                    table[b][j] = None
                taken += 1
        for i in range(n):
            j = (o + i) // page
            if j < len(table[b]) and table[b][j] is not None and cu[b] + i < total:
                slots[cu[b] + i] = table[b][j] * page + (o + i) % page
    return table, slots, [o + cu[b + 1] - cu[b] for b, o in enumerate(old)], taken


@pytest.mark.parametrize("B,page,hi_old,hi_new", [
    (1, 16, 0, 1), (1, 64, 100, 300), (3, 16, 0, 40), (40, 32, 200, 1), (129, 64, 500, 3), (300, 16, 64, 1), (7, 256, 3000, 2000), (5, 1, 9, 9),
])
@pytest.mark.parametrize("seed", [0, 1])
def test_tables_and_slots(B, page, hi_old, hi_new, seed):
    from fold_attention_b200 import decode

    rng = random.Random(seed)
    old = [rng.randint(0, hi_old) for _ in range(B)]
    new = [rng.randint(0, hi_new) if seed else hi_new for _ in range(B)]
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    per = max(1, max(-(-(o + n) // page) for o, n in zip(old, new)))
    pool = sum(-(-(o + n) // page) for o, n in zip(old, new)) + 2
    free = list(range(pool))
    rng.shuffle(free)
    table, taken = [[0] * per for _ in range(B)], 0
    for b, o in enumerate(old):
        for j in range(-(-o // page)):
            table[b][j] = free[taken]
            taken += 1
    want = plain_tables(cu, old, table, page, cu[-1], free, taken)
    t, lens, tk, fr = dev32(table), dev32(old), dev32([taken]), dev32(free)
    for _ in range(2):     # the same call gives the same answer
        slots, after, used = decode.build_tables(dev32(cu), lens, t, page, cu[-1], free_pages=fr, taken=tk)
        assert t.tolist() == want[0] and slots.tolist() == want[1] and after.tolist() == want[2] and used.tolist() == [want[3]]
    assert lens.tolist() == old and tk.tolist() == [taken] and fr.tolist() == free
    # with the table as it now stands, the slots alone
    slots, after, used = decode.build_tables(dev32(cu), lens, t, page, cu[-1])
    assert slots.tolist() == want[1] and after.tolist() == want[2] and used is None


def test_tokens_without_a_place_get_no_slot():
    from fold_attention_b200 import decode

    # two requests, three pages of four left, tables of two pages; five rows more than the requests have
    table = [[9, 0], [8, 0]]
    cu, old = [1, 7, 10], [3, 4]
    slots, lens, used = decode.build_tables(dev32(cu), dev32(old), t := dev32(table), 4, 15, free_pages=dev32([9, 8, 7]), taken=dev32([2]))
    assert slots.tolist() == [-1, 39, 28, 29, 30, 31, -1, -1, -1, -1, -1, -1, -1, -1, -1]
    assert lens.tolist() == [9, 7] and used.tolist() == [5]     # request 0 wants pages 2 and 3 of a table of two, request 1 a page that is not there
    assert t.tolist() == [[9, 7], [8, 0]]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("v8", [False, True])
@pytest.mark.parametrize("n,HKV,page", [(1, 1, 16), (5, 3, 32), (257, 2, 64), (1000, 8, 128), (33, 20, 256)])
def test_tokens_into_the_pool_and_back(dtype, D, v8, n, HKV, page):
    from fold_attention_b200 import decode

    g = torch.Generator(device="cuda").manual_seed(n)
    pages = -(-n // page) + 2
    evs = 0.25 if v8 else 1.0
    # strided: heads and tokens of a wider tensor
    wide = (torch.randn(n, 2 * HKV + 1, D, device="cuda", generator=g) * 3).to(dtype)
    k, v = wide[:, :HKV], wide[:, HKV:2 * HKV]
    slots = torch.randperm(pages * page, device="cuda", generator=g)[:n].int()
    if n > 4:
        slots[3] = -1
    rows = pages * page * HKV
    vdt = torch.float8_e4m3fn if v8 else torch.bfloat16
    ka, kb = (torch.zeros(rows, D, device="cuda", dtype=torch.int8) for _ in range(2))
    va = torch.zeros(rows, D, device="cuda", dtype=vdt)
    vb = torch.zeros(rows, D, device="cuda", dtype=vdt) if v8 else None
    ek = torch.zeros(rows, device="cuda", dtype=torch.bfloat16)
    decode.write_tokens(k, v, slots, page, ka, kb, va, vb, ek, v_scale=evs)
    want = dict(ka=np.zeros((rows, D), np.int8), kb=np.zeros((rows, D), np.int8), ek=np.zeros(rows, np.float32),
                va=np.zeros((rows, D), np.uint8 if v8 else np.float32), vb=np.zeros((rows, D), np.uint8) if v8 else None)
    s = slots.cpu().numpy().astype(np.int64)
    keep = s >= 0
    row = ((s[keep] // page)[:, None] * HKV + np.arange(HKV)) * page + (s[keep] % page)[:, None]
    kf, vf = k.float().cpu().numpy()[keep], v.float().cpu().numpy()[keep]
    stored = vf if v8 else torch.from_numpy(vf).bfloat16().float().numpy()      # the pool is bf16: an fp16 token is rounded to it once
    cf.write_rows(want, kf, stored, evs, row, s[keep] % page)
    assert np.array_equal(ka.cpu().numpy(), want["ka"]) and np.array_equal(kb.cpu().numpy(), want["kb"])
    assert np.array_equal(ek.float().cpu().numpy(), want["ek"])
    bits = (lambda t: t.view(torch.uint8).cpu().numpy()) if v8 else (lambda t: t.float().cpu().numpy())
    assert np.array_equal(bits(va), want["va"]) and (vb is None or np.array_equal(bits(vb), want["vb"]))
    # and back
    pa, pb, e = cf.key_planes(kf)
    val = (pa.astype(np.float64) + pb.astype(np.float64) / 256) * e[..., None].astype(np.float64)
    had = np.ones((1, 1))
    while had.shape[0] < D:
        had = np.block([[had, had], [had, -had]])
    val = torch.from_numpy(val @ had / np.sqrt(D))
    if v8:
        a, b = cf.e4m3_planes(vf, evs)
        back = torch.from_numpy((cf.e4m3_decode(a).astype(np.float64) + cf.e4m3_decode(b).astype(np.float64) / 8) * evs)
    else:
        back = torch.from_numpy(vf).bfloat16().double()
    for dt in (torch.float32, torch.bfloat16, torch.float16):
        kr, vr = decode.read_tokens(slots, page, HKV, ka, kb, va, vb, ek, v_scale=evs, dtype=dt)
        assert kr.shape == (n, HKV, D) and kr.dtype == dt
        assert not kr.cpu()[~torch.from_numpy(keep)].any() and not vr.cpu()[~torch.from_numpy(keep)].any()
        kd, vd = kr.cpu()[torch.from_numpy(keep)].double(), vr.cpu()[torch.from_numpy(keep)].double()
        half = torch.finfo(dt).eps / 2
        tiny = torch.finfo(dt).tiny * half      # below the normal range fp16's steps do not shrink
        lim = 8 * 2.0 ** -24 * val.norm(dim=-1, keepdim=True) + (0 if dt == torch.float32 else half * val.abs()) + tiny
        assert ((kd - val).abs() <= lim).all()
        assert ((vd - back).abs() <= (0 if dt == torch.float32 else half * back.abs()) + tiny).all()


def test_on_another_stream_and_from_a_graph():
    from fold_attention_b200 import decode

    lens, table, cu = dev32([5, 0]), dev32([[0, 0], [0, 0]]), dev32([0, 3, 20])
    free, taken = dev32([6, 4, 2, 0]), dev32([0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            slots, after, used = decode.build_tables(cu, lens, table, 16, 20, free_pages=free, taken=taken)
    lens.copy_(dev32([16, 1]))
    g.replay()
    torch.cuda.synchronize()
    want = plain_tables([0, 3, 20], [16, 1], [[0, 0], [0, 0]], 16, 20, [6, 4, 2, 0], 0)
    assert (table.tolist(), slots.tolist(), after.tolist(), used.tolist()) == (want[0], want[1], want[2], [want[3]])


def test_a_slot_beyond_the_pool_is_no_place():
    from fold_attention_b200 import decode

    HKV, D, page, pages = 3, 64, 16, 2
    rows = pages * page * HKV
    ka, kb = (torch.zeros(rows, D, device="cuda", dtype=torch.int8) for _ in range(2))
    va, ek = torch.zeros(rows, D, device="cuda", dtype=torch.bfloat16), torch.zeros(rows, device="cuda", dtype=torch.bfloat16)
    k = torch.randn(4, HKV, D, device="cuda").bfloat16()
    slots = dev32([31, 32, 2 ** 31 - 1, -2 ** 31])        # the pool's last one, then three that it does not have
    decode.write_tokens(k, k, slots, page, ka, kb, va, None, ek)
    kr, vr = decode.read_tokens(slots, page, HKV, ka, kb, va, None, ek)
    assert torch.equal(vr[0], k[0]) and not vr[1:].any() and not kr[1:].any()
    assert int((ek != 0).sum()) == HKV


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_tokens_off_a_16_byte_boundary(dtype):
    from fold_attention_b200 import decode

    HKV, D, page, n = 2, 64, 16, 5
    k, v = (torch.randn(n, HKV, D, device="cuda").to(dtype) for _ in range(2))
    slots, pools = dev32([3, 17, 0, 30, 9]), []
    for shift in (0, 1):
        ka, kb = (torch.zeros(2 * page * HKV, D, device="cuda", dtype=torch.int8) for _ in range(2))
        va, ek = torch.zeros_like(ka, dtype=torch.bfloat16), torch.zeros(2 * page * HKV, device="cuda", dtype=torch.bfloat16)
        ins = []
        for x in (k, v):
            flat = torch.empty(x.numel() + shift, device="cuda", dtype=dtype)
            flat[shift:] = x.flatten()
            ins.append(flat[shift:].view(x.shape))
        decode.write_tokens(*ins, slots, page, ka, kb, va, None, ek)
        pools.append((ka, kb, va, ek))
    assert all(torch.equal(a, b) for a, b in zip(*pools))
