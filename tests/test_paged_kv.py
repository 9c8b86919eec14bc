"""The paged key-value operators (gguf_kv_*, through the Python binding and,
for refusals, the C-ABI) against their definitions in 64 bits.

Tolerances, per value, from the arithmetic alone:

* a result rounded once to its type: eps / 2 of its magnitude;
* append: the norm's factor is 1 / sqrt of a sum of n squares in fp32, off by
  at most (n / 2 + 4) steps of 2^-24, and the rotation's two products, their
  sum, the cosine and the sine add at most 8 steps of the pair's length;
* attention: a score is off by at most (size + 4) steps of 2^-24 of sum
  |q k| scale =: S, which moves a weight by that much relative to itself (and
  the largest one too, hence twice); the weights' sum and the output's by a
  step per position added; the split of a weight over two values of the
  cache's type leaves 2^-16 (bf16) or 2^-21 (f16) of it; exp2 and the
  division two steps.  All of it times the largest |v|.
"""
import ctypes as C
import math
import random

import numpy as np
import pytest

import vireo_b200 as V

gpu = pytest.mark.gpu
STEP = 2.0 ** -24
F32, F16, BF16 = "float32", "float16", "bfloat16"
PAIRS = [(F32, F32), (F32, F16), (F16, F16), (BF16, BF16)]


def dt(name):
    import torch
    return getattr(torch, name)


def half_eps(dtype):
    import torch
    return torch.finfo(dtype).eps / 2


# ---------------------------------------------------------------------------
# refusals: host checks, no device needed
# ---------------------------------------------------------------------------

def kv_desc(**over):
    f = dict(n_heads=8, n_kv_heads=2, head_size=64, page_size=16, n_pages=4, kv_type=1, act_type=0, k=4096, v=8192,
             page_stride=2 * 16 * 64, head_stride=16 * 64, pos_stride=64, eps=1e-6, rope_base=1e4, rope_dim=64)
    f.update(over)
    return V.GgufKvDesc(**f)


def create(desc):
    h = C.c_void_p()
    st = V._kv_api().gguf_kv_create(C.byref(desc) if desc is not None else None, C.byref(h))
    return st, h


@pytest.mark.parametrize("over,status", [
    (dict(n_heads=0), -1), (dict(n_heads=7), -1), (dict(n_kv_heads=0), -1), (dict(k=None), -1), (dict(v=None), -1),
    (dict(k=4100), -1), (dict(n_pages=0), -1), (dict(eps=-1.0), -1), (dict(eps=float("nan")), -1),
    (dict(rope_base=0.0), -1), (dict(rope_dim=80), -1), (dict(rope_dim=-16), -1), (dict(page_stride=32), -1),
    (dict(pos_stride=65), -1), (dict(head_stride=0), -1), (dict(page_stride=1 << 40), -1),
    (dict(head_size=96, pos_stride=96), -3), (dict(page_size=12), -3), (dict(page_size=4), -3),
    (dict(page_size=2048, head_stride=2048 * 64, page_stride=2 * 2048 * 64), -3), (dict(rope_dim=24), -3),
    (dict(kv_type=8), -3), (dict(kv_type=30, act_type=0), -3), (dict(kv_type=0, act_type=1), -3)])
def test_create_refuses(over, status):
    st, h = create(kv_desc(**over))
    assert st == status and not h.value


def test_create_is_host_only_and_null_calls_are_refused():
    L = V._kv_api()
    assert create(None)[0] == -1
    st, h = create(kv_desc())
    assert st == 0 and h.value
    try:
        assert L.gguf_kv_append(h, None, None) == -1
        assert L.gguf_kv_append(None, C.byref(V.GgufKvAppendArgs()), None) == -1
        assert L.gguf_kv_attn(h, None, None) == -1
        assert L.gguf_kv_attn_topk(h, C.byref(V.GgufKvAttnArgs()), None, None) == -1
        assert L.gguf_kv_plan(None, None) == -1
        assert L.gguf_kv_workspace(None, 1, 1, 0) == 0 and L.gguf_kv_workspace(h, 1, 0, 0) == 0
        assert L.gguf_kv_workspace(h, 4, 8, 0) > 0
        assert L.gguf_kv_workspace(h, 4, 8, 3) > L.gguf_kv_workspace(h, 4, 8, 0)
    finally:
        L.gguf_kv_destroy(h)


APPEND_OK = dict(n_tokens=2, q=4096, k=4096, v=4096, q_stride=512, k_stride=128, v_stride=128, q_out=4096,
                 q_out_stride=512, pos=4096, slots=4096)


@pytest.mark.parametrize("over", [
    dict(n_tokens=-1), dict(q=None), dict(k=4104), dict(q_stride=256), dict(q_stride=513), dict(k_stride=0),
    dict(q_out=None), dict(q_out_stride=511), dict(pos=None), dict(slots=None), dict(means=4104),
    dict(q_norm=4096, q_norm_len=63), dict(k_norm=4096, k_norm_len=512), dict(bq=4100),
    dict(q_norm=4104, q_norm_len=64)])
def test_append_refuses(over):
    L = V._kv_api()
    st, h = create(kv_desc())
    try:
        f = dict(APPEND_OK)
        f.update(over)
        assert L.gguf_kv_append(h, C.byref(V.GgufKvAppendArgs(**f)), None) == -1
    finally:
        L.gguf_kv_destroy(h)


@pytest.mark.parametrize("over", [
    dict(n_seqs=-1), dict(max_pages=0), dict(max_pages=1 << 28), dict(q=None), dict(q=4104), dict(out=None),
    dict(q_stride=500), dict(out_stride=510), dict(table=None), dict(table_stride=7), dict(kv_len=None), dict(ws=None),
    dict(ws=4096 + 16), dict(ws_bytes=100), dict(scale=float("nan")),
    dict(scale=1e300), dict(out_stride=1024)])
def test_attn_refuses(over):
    L = V._kv_api()
    st, h = create(kv_desc())
    try:
        f = dict(n_seqs=2, max_pages=8, q=4096, q_stride=512, out=4096, out_stride=512, table=4096, table_stride=8,
                 kv_len=4096, scale=0.0, ws=4096, ws_bytes=1 << 30)
        f.update(over)
        a = V.GgufKvAttnArgs(**f)
        assert L.gguf_kv_attn(h, C.byref(a), None) == -1
        s = V.GgufKvSelectArgs(4096, 1, 1, 2, None)
        assert L.gguf_kv_attn_topk(h, C.byref(a), C.byref(s), None) == -1
    finally:
        L.gguf_kv_destroy(h)


@pytest.mark.parametrize("sel", [(None, 1, 1, 1), (4104, 1, 1, 1), (4096, -1, 1, 1), (4096, 1, 0, 1), (4096, 1, 1, -1),
                                 (4096, 1 << 30, 1 << 30, 1)])
def test_topk_refuses(sel):
    L = V._kv_api()
    st, h = create(kv_desc())
    try:
        a = V.GgufKvAttnArgs(n_seqs=2, max_pages=8, q=4096, q_stride=512, out=4096, out_stride=512, table=4096,
                             table_stride=8, kv_len=4096, scale=0.0, ws=4096, ws_bytes=1 << 62)
        assert L.gguf_kv_attn_topk(h, C.byref(a), C.byref(V.GgufKvSelectArgs(*sel, None)), None) == -1
    finally:
        L.gguf_kv_destroy(h)


PLAN_OK = dict(n_seqs=2, page_size=16, n_pages=8, max_pages=4, n_slots=4, table_stride=4, past=4096, add=4096,
               table=4096, ring=4096, state=4096, slots=4096, pos=4096, cu=4096, kv_len=4096, granted=4096,
               state_out=4096)


@pytest.mark.parametrize("over,status", [
    (dict(n_seqs=-1), -1), (dict(n_slots=-1), -1), (dict(n_pages=0), -1), (dict(max_pages=0), -1),
    (dict(table_stride=3), -1), (dict(past=None), -1), (dict(ring=None), -1), (dict(state=None), -1),
    (dict(cu=None), -1), (dict(slots=None), -1), (dict(state_out=None), -1),
    (dict(max_pages=1 << 28, table_stride=1 << 28), -1),
    (dict(page_size=0), -1), (dict(page_size=24), -3), (dict(n_seqs=8193), -3)])
def test_plan_refuses(over, status):
    f = dict(PLAN_OK)
    f.update(over)
    assert V._kv_api().gguf_kv_plan(C.byref(V.GgufKvPlanArgs(**f)), None) == status


def test_packed_arguments_have_the_structures_layout():
    import ctypes
    for pack, st in ((V._PLAN_PACK, V.GgufKvPlanArgs), (V._APPEND_PACK, V.GgufKvAppendArgs),
                     (V._ATTN_PACK, V.GgufKvAttnArgs), (V._SELECT_PACK, V.GgufKvSelectArgs)):
        vals = [i + 1.5 if t is C.c_float else i + 1 for i, (_, t) in enumerate(st._fields_)]
        raw = pack(*vals)
        assert len(raw) == ctypes.sizeof(st)
        back = st.from_buffer_copy(raw)
        assert [getattr(back, n) for n, _ in st._fields_] == vals


def test_binding_refuses_host_tensors():
    import torch
    z = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(V.VireoError):
        V.kv_plan(z, z, z.view(4, 1), z, z[:2], 16, slots=z.long(), pos=z, cu=torch.zeros(5, dtype=torch.int32),
                  kv_len=z, granted=z, state_out=z[:2])
    p = torch.zeros(2, 1, 16, 64)
    with pytest.raises(V.VireoError):
        V.PagedKV(p, p.clone(), 4)


def test_binding_refuses_what_no_argument_holds():
    for pack, values in ((V._PLAN_PACK, [1, 2 ** 31] + [1] * 15), (V._SELECT_PACK, [4096, 1, 1, -2 ** 31 - 1, 0]),
                         (V._ATTN_PACK, [1, 2 ** 31] + [1] * 10)):
        with pytest.raises(V.VireoError):
            V._kv_pack(pack, *values)


def test_binding_refuses_a_second_device(monkeypatch):
    import torch

    class Lib:  # a library that works on device 0
        vireo_device_init = staticmethod(lambda dev: 0 if dev == 0 else -1)
    monkeypatch.setattr(V, "lib", lambda: Lib)
    monkeypatch.setattr(V, "_kv_dev", None)
    back = []
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 5)
    monkeypatch.setattr(torch.cuda, "set_device", back.append)
    V._kv_device(0)
    V._kv_device(0)
    assert V._kv_dev == 0 and back == [5]
    with pytest.raises(V.VireoError):
        V._kv_device(1)
    assert V._kv_dev == 0 and back == [5, 5]


# ---------------------------------------------------------------------------
# block tables and slot maps
# ---------------------------------------------------------------------------

def plain_plan(past, add, table, ring, state, page, n_slots):
    """gguf_kv_plan's definition, request by request, on lists (table and ring are changed)."""
    width, n_pages = len(table[0]) if table else 0, len(ring)
    head, count = state
    need_sum = ask_sum = taken = given = 0
    slots, pos, cu, kv_len, granted = [], [], [0], [], []
    free = [ring[(head + j) % n_pages] for j in range(count)]
    for i, (p, a) in enumerate(zip(past, add)):
        have, want = -(-p // page), -(-(p + max(a, 0)) // page)
        ok = p >= 0 and a >= -1 and want <= width
        got = 0
        if ok:
            need_sum += want - have
            ask_sum += max(a, 0)
            ok = (want == have or need_sum <= count) and (a <= 0 or ask_sum <= n_slots)
        if ok and a < 0:
            for j in range(have):
                ring[(head + count + given) % n_pages] = table[i][j]
                given += 1
        elif ok:
            got = a
            for j in range(have, want):
                table[i][j] = free[taken]
                taken += 1
            for j in range(p, p + a):
                pos.append(j)
                slots.append(table[i][j // page] * page + j % page)
        granted.append(int(ok))
        kv_len.append(0 if ok and a < 0 else max(p + got, 0))
        cu.append(cu[-1] + got)
    rest = n_slots - len(slots)
    return (table, ring, slots + [-1] * rest, pos + [0] * rest, cu, kv_len, granted,
            [(head + taken) % n_pages, count - taken + given])


def plan_case(n, page, width, seed, tight):
    r = random.Random(seed)
    past = [r.choice([0, 1, page - 1, page, page + 1, r.randrange(width * page + 1)]) for _ in range(n)]
    past = [min(p, width * page) for p in past]
    add = [r.choice([0, 1, 1, 1, -1, r.randrange(1, 3 * page)]) for _ in range(n)]
    for i in range(0, n, 11):
        past[i], add[i] = r.choice([(-5, 1), (3, -2), (width * page, 1), (page, width * page), (width * page + 1, -1),
                                    (5, 2 ** 31 - 1)])
    used = sum(min(-(-max(p, 0) // page), width) for p in past)
    spare = sum(max(a, 0) for a in add if a < 10 ** 6) // page // (3 if tight else 1) + (0 if tight else 2 * n)
    n_pages = used + spare + 1
    ids = list(range(n_pages))
    r.shuffle(ids)
    table = [[-7] * width for _ in range(n)]
    for row, p in zip(table, past):
        for j in range(min(-(-max(p, 0) // page), width)):
            row[j] = ids.pop()
    head = r.randrange(n_pages)
    ring = [-3] * n_pages
    for j, p in enumerate(ids):
        ring[(head + j) % n_pages] = p
    tokens = sum(a for a in add if 0 < a < 10 ** 6)
    n_slots = tokens // 2 if tight == 2 else tokens + r.choice([0, 37])
    return past, add, table, ring, [head, len(ids)], n_slots


@gpu
@pytest.mark.parametrize("n,page,width,tight", [
    (1, 16, 4, 0), (3, 8, 9, 0), (64, 16, 40, 0), (64, 16, 40, 1), (1000, 32, 33, 2), (1025, 8, 20, 1),
    (8192, 16, 12, 0), (2, 1024, 3, 0)])
def test_plan_matches_the_definition(n, page, width, tight):
    import torch
    past, add, table, ring, state, n_slots = plan_case(n, page, width, 100 * n + tight, tight)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
    wide = torch.full((n, width + 3), -9, dtype=torch.int32, device="cuda")
    t = wide[:, :width]
    t.copy_(i32(table))
    pa, ri = i32(past), i32(ring)
    new = lambda k, d=torch.int32: torch.full((k,), 99, dtype=d, device="cuda")
    slots, pos, cu, kv, gr, so = new(n_slots, torch.int64), new(n_slots), new(n + 1), new(n), new(n), new(2)
    for _ in range(2):  # a repeated call repeats its results
        V.kv_plan(pa, i32(add), t, ri, i32(state), page, slots=slots, pos=pos, cu=cu, kv_len=kv, granted=gr,
                  state_out=so)
    got = [x.cpu().tolist() for x in (t, ri, slots, pos, cu, kv, gr, so)]
    want = plain_plan(past, add, table, ring, state, page, n_slots)
    for name, a, b in zip(("table", "ring", "slots", "pos", "cu", "kv_len", "granted", "state"), got, want):
        assert a == b, name
    assert (wide[:, width:] == -9).all()


@gpu
@pytest.mark.parametrize("n,page,width,tight,what", [
    (64, 16, 40, 1, "both"), (1000, 32, 33, 2, "both"), (1000, 8, 20, 0, "kv_len"), (1025, 8, 20, 1, "state"),
    (8192, 16, 12, 0, "both")])
def test_plan_in_place_matches_the_definition(n, page, width, tight, what):
    """Lengths, state or both updated in place, by one CTA and by several, three calls in a row."""
    import torch
    past, add, table, ring, state, n_slots = plan_case(n, page, width, 7 * n + tight, tight)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
    new = lambda k, d=torch.int32: torch.full((k,), 99, dtype=d, device="cuda")
    t, ri, a, pa, s = i32(table), i32(ring), i32(add), i32(past), i32(state)
    slots, pos, cu, gr = new(n_slots, torch.int64), new(n_slots), new(n + 1), new(n)
    for _ in range(3):
        kv = pa if what != "state" else new(n)
        so = s if what != "kv_len" else new(2)
        V.kv_plan(pa, a, t, ri, s, page, slots=slots, pos=pos, cu=cu, kv_len=kv, granted=gr, state_out=so)
        want = plain_plan(past, add, table, ring, state, page, n_slots)
        got = [x.cpu().tolist() for x in (t, ri, slots, pos, cu, kv, gr, so)]
        for name, x, y in zip(("table", "ring", "slots", "pos", "cu", "kv_len", "granted", "state"), got, want):
            assert x == y, name
        table, ring, past, state, pa, s = want[0], want[1], want[5], want[7], kv, so


@gpu
def test_plan_in_place_and_without_requests():
    import torch
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
    kv, state, ring = i32([5, 16, 0]), i32([1, 4]), i32([9, 3, 1, 0, 2, 9])
    table = i32([[4, -1], [5, -1], [-1, -1]])
    slots, pos, cu, gr = torch.zeros(3, dtype=torch.int64).cuda(), i32([0] * 3), i32([0] * 4), i32([0] * 3)
    V.kv_plan(kv, i32([1, 1, -1]), table, ring, state, 16, slots=slots, pos=pos, cu=cu, kv_len=kv, granted=gr,
              state_out=state)
    assert kv.tolist() == [6, 17, 0] and state.tolist() == [2, 3] and slots.tolist() == [4 * 16 + 5, 3 * 16, -1]
    assert table.tolist() == [[4, -1], [5, 3], [-1, -1]] and cu.tolist() == [0, 1, 2, 2] and gr.tolist() == [1, 1, 1]
    none = torch.zeros(0, dtype=torch.int32).cuda()
    slots.fill_(5)
    V.kv_plan(none, none, torch.zeros(0, 2, dtype=torch.int32).cuda(), ring, state, 16, slots=slots, pos=pos,
              cu=cu[:1], kv_len=none, granted=none, state_out=state)
    assert slots.tolist() == [-1] * 3 and state.tolist() == [2, 3] and cu[0].item() == 0


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------

def make_pool(n_pages, g, page, d, dtype, tokens_first, gen, fill=None):
    import torch
    shape = (n_pages, page, g, d) if tokens_first else (n_pages, g, page, d)
    if fill is None:
        x = torch.randn(shape, generator=gen, device="cuda").to(dtype)
    else:
        x = torch.full(shape, fill, device="cuda", dtype=dtype)
    return x.transpose(1, 2) if tokens_first else x


def plain_append_rows(x, bias, w, heads, d, pos, rope, base, eps):
    """[t, heads, d] in 64 bits, and the bound's scale: the pair lengths."""
    import torch
    y = x.double()
    if bias is not None:
        y = y + bias.double()
    y = y.reshape(-1, heads, d)
    if w is not None:
        if w.numel() == d:
            y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
        else:
            y = y / (y.square().mean((1, 2), keepdim=True) + eps).sqrt() * w.double().reshape(heads, d)
    mag = y.abs()
    if pos is not None and rope:
        h = rope // 2
        ang = pos.double()[:, None] * base ** (-2.0 * torch.arange(h, device=x.device, dtype=torch.float64) / rope)
        c, s = ang.cos()[:, None], ang.sin()[:, None]
        a, b = y[..., :h], y[..., h:rope]
        pair = torch.sqrt(a * a + b * b)
        y = torch.cat([a * c - b * s, a * s + b * c, y[..., rope:]], -1)
        mag = torch.cat([pair, pair, mag[..., rope:]], -1)
    return y, mag


APPEND_CASES = [
    # tokens, heads, kv heads, size, (act, kv), page, norm, bias, rope, means, tokens_first
    (1, 16, 16, 128, (F32, F16), 16, "full", False, 128, False, False),
    (5, 8, 1, 64, (F32, F32), 8, "head", True, 64, True, False),
    (37, 14, 2, 64, (F16, F16), 16, "none", True, 32, True, True),
    (130, 32, 4, 128, (BF16, BF16), 64, "head", False, 128, True, False),
    (64, 6, 3, 256, (F32, F32), 32, "full", True, 256, True, True),
    (33, 5, 5, 256, (BF16, BF16), 8, "head", False, 0, True, False),
    (600, 1, 1, 128, (F32, F16), 128, "full", False, 16, True, False),
    (1027, 4, 2, 64, (F16, F16), 1024, "head", False, 64, True, True),
    (700, 12, 4, 256, (F32, F16), 16, "full", True, 256, False, False),
    (1301, 5, 1, 64, (BF16, BF16), 32, "full", True, 32, True, False),
    (2003, 1, 1, 128, (F32, F32), 16, "full", False, 128, False, True),
    (900, 40, 20, 64, (F16, F16), 8, "full", False, 64, True, True),
    (350, 3, 1, 128, (F32, F16), 64, "full", True, 0, False, False),
]


@gpu
@pytest.mark.parametrize("case", APPEND_CASES, ids=str)
def test_append(case):
    import torch
    t, h, g, d, (act, kv), page, norm, bias, rope, means, tf = case
    a, c = dt(act), dt(kv)
    gen = torch.Generator(device="cuda").manual_seed(t)
    r = random.Random(t)
    n_pages = -(-t // page) + 3
    kp, vp = (make_pool(n_pages, g, page, d, c, tf, gen) for _ in range(2))
    k0, v0 = kp.clone(), vp.clone()
    qkv = (torch.randn(t, (h + 2 * g) * d, generator=gen, device="cuda") * 2).to(a)
    q, k, v = qkv[:, :h * d], qkv[:, h * d:(h + g) * d], qkv[:, (h + g) * d:]
    vec = lambda n: torch.randn(n, generator=gen, device="cuda") * 0.3 + 1
    qn = kn = bq = bk = bv = None
    if norm != "none":
        qn, kn = (vec(h * d), vec(g * d)) if norm == "full" else (vec(d), vec(d))
    if bias:
        bq, bk, bv = vec(h * d), vec(g * d), vec(g * d)
    order = list(range(n_pages))
    r.shuffle(order)
    slots = [order[i // page] * page + i % page for i in range(t)]
    skipped = [i for i in range(t) if i % 9 == 4]
    for i in skipped:
        slots[i] = -1
    first = r.choice([0, 5, 100000, 2 ** 30])
    pos = torch.tensor([first + i for i in range(t)], dtype=torch.int32).cuda()
    slot = torch.tensor(slots).cuda()
    q_out = torch.full((t, h * d), 7.0, dtype=a, device="cuda")
    m = torch.full((n_pages, g, d), 5.0, dtype=c, device="cuda") if means else None
    P = V.PagedKV(kp, vp, h, a, eps=1e-5, rope_base=5e5, rope_dim=rope)
    P.append(q, k, v, pos, slot, q_out, q_norm=qn, k_norm=kn, bq=bq, bk=bk, bv=bv, means=m)
    P.sync()
    keep = [i for i in range(t) if slots[i] >= 0]
    ki = torch.tensor(keep).cuda()
    page_of, off = slot[ki] // page, slot[ki] % page

    def near(got, ref, mag, n, dtype):
        tol = half_eps(dtype) * ref.abs() + (n / 2 + 12) * STEP * mag + torch.finfo(dtype).tiny
        bad = (got.double() - ref).abs() > tol
        assert not bad.any(), (int(bad.sum()), float(((got.double() - ref).abs() / tol).max()))

    nq, nk = (h * d, g * d) if norm == "full" else (d, d)
    ref, mag = plain_append_rows(q, bq, qn, h, d, pos, rope, 5e5, 1e-5)
    near(q_out.reshape(t, h, d)[ki], ref[ki], mag[ki], nq, a)
    if skipped:
        assert (q_out[torch.tensor(skipped).cuda()] == 7.0).all()
    ref, mag = plain_append_rows(k, bk, kn, g, d, pos, rope, 5e5, 1e-5)
    near(kp[page_of, :, off], ref[ki], mag[ki], nk, c)
    ref, mag = plain_append_rows(v, bv, None, g, d, None, 0, 1, 0)
    near(vp[page_of, :, off], ref[ki], mag[ki], 0, c)
    # nothing else of the pool
    k0[page_of, :, off] = kp[page_of, :, off]
    v0[page_of, :, off] = vp[page_of, :, off]
    assert torch.equal(kp, k0) and torch.equal(vp, v0)
    if means:
        ends = sorted({s // page for s in slots if s >= 0 and s % page == page - 1})
        for p in range(n_pages):
            if p in ends:
                x = kp[p].double()
                ref = x.mean(1)
                tol = half_eps(c) * ref.abs() + page * STEP * x.abs().mean(1) + torch.finfo(c).tiny
                assert ((m[p].double() - ref).abs() <= tol).all()
            else:
                assert (m[p] == 5.0).all()
    # in place, and in heads
    q2 = qkv.clone()
    P.append(q2[:, :h * d].reshape(t, h, d) if t == 1 else q2[:, :h * d], k, v, pos, slot, q2[:, :h * d], q_norm=qn,
             k_norm=kn, bq=bq, bk=bk, bv=bv)
    assert torch.equal(q2[ki][:, :h * d], q_out[ki])


@gpu
def test_append_bits_do_not_depend_on_the_batch():
    """A token's rows come out the same alone and among others, with per-head
    and with full-width norms."""
    import torch
    gen = torch.Generator(device="cuda").manual_seed(8)
    for h, g, d, act, full in ((5, 1, 64, F16, True), (5, 1, 64, F32, True), (16, 16, 128, F32, True),
                               (40, 20, 64, BF16, True), (32, 4, 128, BF16, False), (6, 2, 256, F32, False)):
        n = 1500
        kp, vp = (torch.zeros(n // 8 + 1, g, 8, d, device="cuda", dtype=dt(act)) for _ in range(2))
        q, k = (torch.randn(n, w * d, generator=gen, device="cuda").to(dt(act)) for w in (h, g))
        qn, kn = (torch.rand(w, generator=gen, device="cuda") for w in ((h * d, g * d) if full else (d, d)))
        pos = torch.arange(n, dtype=torch.int32, device="cuda") * 7
        slots = torch.arange(n, device="cuda")
        P = V.PagedKV(kp, vp, h)
        want = torch.empty_like(q)
        P.append(q, k, k, pos, slots, want, q_norm=qn, k_norm=kn)
        keys = kp.clone()
        for lo, hi in ((0, 1), (7, 8), (100, 117), (600, 1100), (1499, 1500)):
            got = torch.empty_like(q[lo:hi])
            P.append(q[lo:hi], k[lo:hi], k[lo:hi], pos[lo:hi], slots[lo:hi], got, q_norm=qn, k_norm=kn)
            assert torch.equal(got, want[lo:hi]), (h, g, d, act, lo)
            assert torch.equal(kp, keys)


@gpu
@pytest.mark.parametrize("h,g,d,act,kv,q_len,k_len", [
    (16, 16, 128, F32, F16, "full", "full"), (14, 2, 64, F16, F16, "full", "head"), (7, 7, 64, F32, F32, "head", "full"),
    (12, 1, 256, BF16, BF16, "full", None), (64, 8, 128, BF16, BF16, None, "full"),
    (300, 100, 64, BF16, BF16, "full", "full")])
def test_append_of_many_tokens_is_that_of_few(h, g, d, act, kv, q_len, k_len):
    """One call over 1301 tokens gives the bits of calls over 100 each: full
    widths on either side or both, biases, skipped and bad slots, in place."""
    import torch
    n, page = 1301, 16
    gen = torch.Generator(device="cuda").manual_seed(h * d)
    pools = [torch.zeros(n // page + 1, g, page, d, device="cuda", dtype=dt(kv)) for _ in range(4)]
    q, k, v = (torch.randn(n, w * d, generator=gen, device="cuda").to(dt(act)) for w in (h, g, g))
    vec = lambda w: torch.rand(w, generator=gen, device="cuda")
    norm = lambda length, w: {None: None, "full": vec(w * d), "head": vec(d)}[length]
    named = dict(q_norm=norm(q_len, h), k_norm=norm(k_len, g), bq=vec(h * d), bk=vec(g * d), bv=vec(g * d))
    pos = torch.randint(0, 100000, (n,), generator=gen, device="cuda", dtype=torch.int32)
    slots = torch.randperm(n, generator=gen, device="cuda")
    slots[::13] = -1
    one, many = (V.PagedKV(*p, h, dt(act), rope_dim=d // 2) for p in (pools[:2], pools[2:]))
    out = [torch.full_like(q, 3.0) for _ in range(2)]
    one.append(q, k, v, pos, slots, out[0], **named)
    for i in range(0, n, 100):
        j = slice(i, i + 100)
        many.append(q[j], k[j], v[j], pos[j], slots[j], out[1][j], **named)
    one.sync()
    assert torch.equal(out[0], out[1]) and (out[0][::13] == 3.0).all()
    for a, b in ((0, 2), (1, 3)):
        assert torch.equal(pools[a], pools[b]) and pools[a].abs().sum() > 0
    in_place = q.clone()
    in_place[::13] = 3.0
    slots[5] = 2 ** 33
    out[0][5] = in_place[5]
    one.append(in_place, k, v, pos, slots, in_place, **named)
    with pytest.raises(V.VireoError):
        one.sync()
    assert torch.equal(in_place, out[0])


@gpu
def test_append_reports_slots_outside_the_pool():
    import torch
    kp, vp = (torch.zeros(4, 2, 8, 64, device="cuda") for _ in range(2))
    P = V.PagedKV(kp, vp, 2)
    x = torch.randn(3, 128, device="cuda")
    out = torch.full_like(x, 3.0)
    pos = torch.arange(3, dtype=torch.int32, device="cuda")
    P.append(x, x, x, pos, torch.tensor([3, 32, 2 ** 40], device="cuda"), out)
    with pytest.raises(V.VireoError) as e:
        P.sync()
    assert e.value.status == -1
    assert (out[1:] == 3.0).all() and (out[0] != 3.0).any() and kp[0, :, 3].abs().sum() > 0
    kp[0, :, 3] = 0
    assert kp.abs().sum() == 0
    P.sync()  # reported once


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

def plain_attn(q, k, v, scale):
    """One request: q [g, r, d], k and v [g, n, d] in 64 bits; (out, bound's scale S)."""
    w = q @ k.transpose(1, 2) * scale
    s = float((q.abs() @ k.abs().transpose(1, 2)).max()) * abs(scale)
    w = w - w.amax(-1, keepdim=True)
    w = w.exp()
    return w @ v / w.sum(-1, keepdim=True), s


def attn_tol(ref, s, vmax, n, d, act, kv):
    split = {F32: 0.0, F16: 2.0 ** -21, BF16: 2.0 ** -16}[kv]
    return half_eps(dt(act)) * ref.abs() + vmax * ((2 * (d + 4) * s + n + 4) * STEP + split)


def make_requests(lens, h, g, d, act, kv, page, tf, seed, hot=1.0, poison=True):
    """A pool whose unused places hold NaN, tables whose unused entries point nowhere."""
    import torch
    gen = torch.Generator(device="cuda").manual_seed(seed)
    need = [-(-n // page) for n in lens]
    n_pages, width = sum(need) + 2, max(max(need), 1) + 2
    kp, vp = (make_pool(n_pages, g, page, d, dt(kv), tf, gen, math.nan if poison else None) for _ in range(2))
    ids = torch.randperm(n_pages, generator=gen, device="cuda").tolist()
    table = torch.full((len(lens), width), 2 ** 31 - 1, dtype=torch.int32)
    for i, n in enumerate(lens):
        for j in range(need[i]):
            p = ids.pop()
            table[i, j] = p
            k = min(page, n - j * page)
            kp[p, :, :k] = (torch.randn(g, k, d, generator=gen, device="cuda") * hot).to(dt(kv))
            vp[p, :, :k] = torch.randn(g, k, d, generator=gen, device="cuda").to(dt(kv))
    q = (torch.randn(len(lens), h * d, generator=gen, device="cuda") * hot).to(dt(act))
    return kp, vp, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), q


def rows_of(pool, pages, n):
    """[g, n, d] of a request's pages, in 64 bits."""
    x = pool[pages.long()].transpose(0, 1)
    return x.reshape(x.shape[0], -1, x.shape[-1])[:, :n].double()


def check_attn(out, q, kp, vp, table, lens, h, act, kv, scale, page):
    g, d = kp.shape[1], kp.shape[3]
    for i, n in enumerate(lens):
        got = out[i].double().reshape(g, -1, d)
        if n == 0:
            assert (got == 0).all(), i
            continue
        pages = table[i, :-(-n // page)]
        k, v = rows_of(kp, pages, n), rows_of(vp, pages, n)
        ref, s = plain_attn(q[i].double().reshape(g, h // g, d), k, v, scale)
        tol = attn_tol(ref, s, float(v.abs().max()), n, d, act, kv)
        err = (got - ref).abs()
        assert (err <= tol).all(), (i, n, float((err / tol).max()))


ATTN_CASES = [
    # lens, heads, kv heads, size, (act, kv), page, tokens_first, hot
    ([1], 1, 1, 64, (F32, F32), 8, False, 1.0),
    ([300], 16, 16, 128, (F32, F16), 16, False, 1.0),
    ([8200], 32, 4, 128, (F32, F16), 64, False, 1.0),
    ([0, 64, 63, 65, 1, 0, 128, 1000], 28, 4, 64, (F16, F16), 8, True, 1.5),
    ([0, 0, 0], 8, 2, 128, (BF16, BF16), 16, False, 1.0),
    ([5, 2049, 0, 777], 32, 4, 128, (BF16, BF16), 16, False, 2.0),
    ([31, 32, 33, 500, 0], 6, 3, 128, (F32, F32), 32, True, 1.0),
    ([1025, 7], 16, 1, 128, (F32, F32), 1024, False, 1.0),
    ([700, 64], 12, 1, 256, (F16, F16), 32, False, 1.0),
    ([257, 90], 16, 1, 256, (F32, F16), 128, True, 1.0),
    ([129, 1, 640], 10, 2, 256, (BF16, BF16), 8, False, 1.0),
    ([400, 33], 4, 1, 256, (F32, F32), 64, False, 1.0),
    ([400, 33, 1500], 8, 1, 256, (F32, F32), 16, False, 1.0),
    ([700, 0, 90], 22, 2, 256, (F32, F32), 32, True, 1.0),
    ([1200, 77], 7, 1, 128, (F32, F32), 8, True, 1.0),
    ([1, 1, 0, 1], 8, 8, 256, (F32, F32), 8, False, 1.0),
    ([2000, 5, 0, 640], 24, 2, 128, (BF16, BF16), 16, False, 1.0),
    ([3000], 16, 1, 128, (F16, F16), 8, True, 2.0),
    ([1000, 129], 38, 2, 64, (F32, F16), 32, False, 1.0),
    ([400, 90], 18, 1, 128, (F32, F32), 16, False, 1.0),
    ([65, 200], 9, 1, 64, (F32, F16), 16, False, 4.0),
    ([65, 200], 3, 3, 64, (F32, F32), 16, True, 4.0),
    ([90, 200], 40, 2, 64, (F32, F32), 8, False, 1.0),
    ([65, 0, 300, 7], 16, 2, 64, (F32, F32), 16, False, 1.5),
    ([1000], 10, 2, 64, (F32, F32), 8, True, 1.0),
    ([40, 2000], 5, 1, 128, (F32, F32), 32, False, 1.0),
    ([60, 0, 130], 24, 2, 256, (F16, F16), 16, False, 1.0),
    ([50, 9, 0], 40, 1, 128, (F32, F32), 8, True, 1.0),
    ([90, 0, 1] * 60, 20, 5, 64, (F32, F32), 16, False, 1.0),
    ([600] + [3] * 99, 48, 8, 128, (BF16, BF16), 16, False, 1.0),
    ([(37 * i) % 211 for i in range(300)], 4, 2, 64, (BF16, BF16), 16, False, 1.0),
]


@gpu
@pytest.mark.parametrize("case", ATTN_CASES, ids=lambda c: str(c)[-60:])
def test_attn(case):
    import torch
    lens, h, g, d, (act, kv), page, tf, hot = case
    kp, vp, table, kv_len, q = make_requests(lens, h, g, d, act, kv, page, tf, 11, hot)
    P = V.PagedKV(kp, vp, h, dt(act))
    out = torch.full_like(q, math.nan)
    P.attn(q, table, kv_len, out)
    P.sync()
    check_attn(out, q, kp, vp, table, lens, h, act, kv, 1 / math.sqrt(d), page)
    again = torch.full_like(q, 1.0)
    P.attn(q.view(len(lens), h, d), table, kv_len, again.view(len(lens), h, d), scale=1 / math.sqrt(d))
    assert torch.equal(again, out)  # the same bits every time
    # strided rows, another scale, out over q
    wide = torch.zeros(len(lens), h * d + 64, dtype=q.dtype, device="cuda")
    wide[:, :h * d] = q
    P.attn(wide[:, :h * d], table, kv_len, wide[:, :h * d], scale=-0.05)
    check_attn(wide[:, :h * d], q, kp, vp, table, lens, h, act, kv, -0.05, page)
    assert (wide[:, h * d:] == 0).all()


@gpu
@pytest.mark.parametrize("r", [2, 8, 11])
@pytest.mark.parametrize("act,kv", PAIRS)
def test_attn_infinities(act, kv, r):
    """A key of -inf scores takes no weight wherever it stands, also when it
    fills the first tiles; a row of nothing else is zero; one +inf or NaN
    score spoils its own head and request only."""
    import torch
    h, g, d, page, lens = 2 * r, 2, 64, 16, [200, 70, 90, 130]
    kp, vp, table, kv_len, q = make_requests(lens, h, g, d, act, kv, page, False, 5)
    q.copy_(q.abs() + 0.1)
    minus = torch.full((d,), -math.inf, device="cuda")
    for i, bad in ((0, range(0, 130)), (1, range(0, 70))):
        for j in bad:
            kp[table[i, j // page].item(), :, j % page] = minus.to(kp.dtype)
    p2 = table[2, 1].item()
    kp[p2, 1, 3] = math.inf
    vp[table[3, 2].item(), 0, 5, 7] = math.nan
    vp[table[3, 1].item(), 1, 2, 9] = -math.inf
    kp[table[3, 1].item(), 1, 2] = 0.0  # a weight well above zero
    P = V.PagedKV(kp, vp, h, dt(act))
    out = torch.full_like(q, 9.0)
    P.attn(q, table, kv_len, out)
    P.sync()
    # request 0: as if the first 130 positions were not there
    k, v = rows_of(kp, table[0, :13], 200)[:, 130:], rows_of(vp, table[0, :13], 200)[:, 130:]
    ref, s = plain_attn(q[0].double().reshape(g, r, d), k, v, 1 / math.sqrt(d))
    err = (out[0].double().reshape(g, r, d) - ref).abs()
    assert (err <= attn_tol(ref, s, float(v.abs().max()), 200, d, act, kv)).all()
    assert (out[1] == 0).all()
    two, three = out[2].reshape(g, r, d), out[3].reshape(g, r, d)
    assert two[0].isfinite().all() and two[1].isnan().all()
    assert (three[1, :, 9] == -math.inf).all() and three[0, :, 7].isnan().all()
    for a, skip in ((0, 7), (1, 9)):
        assert three[a, :, [j for j in range(d) if j != skip]].isfinite().all()


@gpu
@pytest.mark.parametrize("act,kv,d,page", [(F32, F16, 64, 8), (BF16, BF16, 128, 64), (F32, F32, 64, 32)])
def test_attn_bad_pages_and_lengths_are_reported(act, kv, d, page):
    """A page number outside the pool reads as zero keys and values, a length
    beyond the table is cut; both are reported, once."""
    import torch
    lens = [3 * page, 3 * page, 2 * page + 1]
    kp, vp, table, kv_len, q = make_requests(lens, 4, 2, d, act, kv, page, False, 3)
    P = V.PagedKV(kp, vp, 4, dt(act))
    table = table[:, :3].contiguous()
    table[0, 1], table[1, 2] = -1, kp.shape[0]
    kv_len[2] = 2 ** 31 - 1
    table[2, 2] = table[0, 0]
    out = torch.empty_like(q)
    P.attn(q, table, kv_len, out)
    with pytest.raises(V.VireoError) as e:
        P.sync()
    assert e.value.status == -1
    zk = torch.cat([kp, torch.zeros_like(kp[:1])]), torch.cat([vp, torch.zeros_like(vp[:1])])
    t2 = table.clone()
    t2[0, 1] = t2[1, 2] = kp.shape[0]
    check_attn(out[:2], q[:2], *zk, t2[:2], lens[:2], 4, act, kv, 1 / math.sqrt(d), page)
    kv_len[2] = 3 * page
    again = torch.empty_like(q)
    P2 = V.PagedKV(*zk, 4, dt(act))
    P2.attn(q, t2, kv_len, again)
    P2.sync()
    assert torch.equal(again, out)
    kv_len.fill_(-4)
    P2.attn(q, t2, kv_len, again)
    P2.sync()
    assert (again == 0).all()


# ---------------------------------------------------------------------------
# attention over selected pages
# ---------------------------------------------------------------------------

def plain_select(q, means, n, page, sink, window, top):
    """Chosen pages of one request and kv head: q [r, d], means [pages, d]."""
    total = -(-n // page)
    if total <= sink + window + top:
        return list(range(total))
    s = np.asarray(q, np.float64) @ np.asarray(means, np.float64).T
    s = np.where(np.isnan(s), -np.inf, s).max(0)
    mid = sorted(range(sink, total - window), key=lambda p: (-s[p], p))[:top]
    return sorted(list(range(sink)) + mid + list(range(total - window, total)))


def run_topk(lens, h, g, d, act, kv, page, tf, sink, window, top, seed, means=None, quant=False, change_q=None):
    import torch
    kp, vp, table, kv_len, q = make_requests(lens, h, g, d, act, kv, page, tf, seed, poison=True)
    if change_q:
        change_q(q)
    if means is not None:
        means = means(kp.shape[0])
    else:
        means = torch.full((kp.shape[0], g, d), math.nan, device="cuda", dtype=kp.dtype)
        for i, n in enumerate(lens):
            for j in range(n // page):
                p = table[i, j].item()
                means[p] = kp[p].float().mean(1).to(kp.dtype)
        if quant:  # few distinct values, small whole numbers: many exact ties
            means = torch.where(means.isnan(), means, (means * 2).round().clamp(-1, 1))
            q.copy_((q * 1.5).round().clamp(-2, 2))
    P = V.PagedKV(kp, vp, h, dt(act))
    ns = sink + window + top
    sel = torch.full((len(lens), g, ns), 77, dtype=torch.int32, device="cuda")
    out = torch.full_like(q, math.nan)
    P.attn_topk(q, table, kv_len, means, sink, window, top, out, sel=sel)
    P.sync()
    r = h // g
    for i, n in enumerate(lens):
        total = -(-n // page)
        for a in range(g):
            qs = q[i].reshape(g, r, d)[a].double().cpu().numpy()
            ms = means[table[i, :total].long(), a].double().cpu().numpy() if total else np.zeros((0, d))
            want = plain_select(qs, ms, n, page, sink, window, top)
            got = sel[i, a].tolist()
            assert got == want + [-1] * (ns - len(want)), (i, a, n)
            if n == 0:
                assert (out[i] == 0).all()
                continue
            at = torch.tensor([j for p in want for j in range(p * page, min(n, (p + 1) * page))]).cuda()
            pg = table[i].long()[at // page]
            k, v = kp[pg, a, at % page].double()[None], vp[pg, a, at % page].double()[None]
            ref, s = plain_attn(q[i].reshape(g, r, d)[a].double()[None], k, v, 1 / math.sqrt(d))
            err = (out[i].double().reshape(g, r, d)[a] - ref[0]).abs()
            tol = attn_tol(ref[0], s, float(v.abs().max()), at.numel(), d, act, kv)
            assert (err <= tol).all(), (i, a, n, float((err / tol).max()))
    again = torch.empty_like(out)
    P.attn_topk(q, table, kv_len, means, sink, window, top, again)  # without sel
    assert torch.equal(again, out)


TOPK_CASES = [
    # lens, heads, kv heads, size, (act, kv), page, tokens_first, sink, window, top
    ([1], 1, 1, 64, (F32, F32), 8, False, 0, 1, 1),
    ([2000], 32, 4, 128, (BF16, BF16), 16, False, 1, 4, 20),
    ([0, 5, 64, 65, 200, 1000, 513], 8, 2, 64, (F16, F16), 8, True, 2, 2, 5),
    ([900, 300], 12, 1, 256, (F32, F16), 32, False, 0, 1, 3),
    ([700, 701], 20, 2, 128, (F32, F32), 16, True, 3, 1, 0),
    ([640], 6, 6, 64, (F32, F16), 64, False, 0, 3, 4),
    ([5000, 0, 8191], 4, 1, 64, (BF16, BF16), 8, False, 1, 1, 600),
    ([3001, 200], 16, 1, 256, (F32, F32), 16, True, 2, 3, 30),
    ([20000, 9], 2, 1, 256, (BF16, BF16), 8, True, 0, 1, 1),
    ([2600], 7, 1, 128, (F16, F16), 8, False, 4, 2, 77),
    ([70000, 5], 3, 1, 64, (F16, F16), 8, False, 2, 1, 900),
    ([1500, 80], 20, 1, 64, (F32, F32), 8, False, 1, 1, 40),
    ([700, 0, 1300], 34, 2, 256, (BF16, BF16), 16, False, 0, 2, 7),
    ([4000], 33, 1, 128, (F32, F16), 16, True, 2, 1, 30),
]


@gpu
@pytest.mark.parametrize("case", TOPK_CASES, ids=lambda c: str(c)[-60:])
def test_topk(case):
    lens, h, g, d, (act, kv), page, tf, sink, window, top = case
    run_topk(lens, h, g, d, act, kv, page, tf, sink, window, top, 21)


@gpu
@pytest.mark.parametrize("lens,page,top", [([3000], 8, 17), ([2500, 90], 16, 3), ([40000], 8, 300), ([70000], 8, 2000)])
def test_topk_ties_go_to_the_lower_page(lens, page, top):
    run_topk(lens, 4, 2, 64, F32, F16, page, False, 1, 2, top, 8, quant=True)


@gpu
@pytest.mark.parametrize("top", [3, 60, 500])
@pytest.mark.parametrize("shape", ["one far above", "clusters", "negative", "tiny", "infinite", "equal but one"])
def test_topk_of_unusual_scores(shape, top):
    """Scores of every spread: far apart, in clusters, all negative, subnormal
    as fp32, with infinities, all alike."""
    import torch
    gen = torch.Generator(device="cuda").manual_seed(top)

    def means(n):
        x = torch.randn(n, 2, 64, generator=gen, device="cuda").abs()
        row = torch.arange(n, device="cuda").view(n, 1, 1)
        if shape == "one far above":
            x = torch.where(row == 7, 1e6 * x, x * 1e-3)
        elif shape == "clusters":
            x = x * 2.0 ** -(row % 5 * 12).float()
        elif shape == "negative":
            x = -x
        elif shape == "tiny":
            x = x * 1e-40
        elif shape == "infinite":
            x = torch.where(row % 50 == 3, math.inf, x)
        else:
            x = torch.where(row == 11, 1.5, torch.ones_like(x))
        return x

    def positive(q):
        q.abs_()
    run_topk([6000, 40, 2500], 4, 2, 64, F32, F32, 8, False, 1, 2, top, 31, means=means, change_q=positive)


@gpu
def test_topk_scores_of_infinity_nan_and_signed_zero():
    import torch
    n, page = 20 * 8 + 3, 8
    kp, vp, table, kv_len, q = make_requests([n], 2, 1, 64, F32, F32, page, False, 2)
    q.zero_()
    q[0, 0] = 1.0  # scores of the first head: the means' first value; of the second: zero
    q[0, 64] = -1.0
    means = torch.zeros(kp.shape[0], 1, 64, device="cuda")
    vals = [0.0, -0.0, math.nan, math.inf, -math.inf, 3.0, -3.0, 1e-40, 3.0] + [0.0] * 12
    for j, x in enumerate(vals):
        means[table[0, j].item(), 0, 0] = x
    P = V.PagedKV(kp, vp, 2)
    sel = torch.zeros(1, 1, 7, dtype=torch.int32, device="cuda")
    out = torch.empty_like(q)
    P.attn_topk(q, table, kv_len, means, 0, 1, 6, out, sel=sel)
    P.sync()
    # a page's score is |value| here (the larger of value and -value); no
    # inf * 0, since the means' other values are zero and not infinite
    assert sel[0, 0].tolist() == [3, 4, 5, 6, 7, 8, 20]
    assert out.isfinite().all()
    sel = torch.zeros(1, 1, 9, dtype=torch.int32, device="cuda")
    P.attn_topk(q, table, kv_len, means, 0, 1, 8, out, sel=sel)
    assert sel[0, 0].tolist() == [0, 1, 3, 4, 5, 6, 7, 8, 20]
    sel = torch.zeros(1, 1, 20, dtype=torch.int32, device="cuda")
    P.attn_topk(q, table, kv_len, means, 0, 1, 19, out, sel=sel)
    assert sel[0, 0].tolist() == [0, 1] + list(range(3, 21))  # the NaN last of all


@gpu
def test_topk_with_room_for_every_page_is_attention():
    import torch
    lens = [100, 0, 333]
    kp, vp, table, kv_len, q = make_requests(lens, 8, 2, 128, BF16, BF16, 16, False, 4)
    means = torch.full((kp.shape[0], 2, 128), math.nan, device="cuda", dtype=torch.bfloat16)
    P = V.PagedKV(kp, vp, 8)
    a, b = torch.empty_like(q), torch.empty_like(q)
    P.attn(q, table, kv_len, a)
    P.attn_topk(q, table, kv_len, means, 3, 8, 20, b)
    assert torch.equal(a, b)


# ---------------------------------------------------------------------------
# how the calls are made
# ---------------------------------------------------------------------------

@gpu
def test_far_pages_of_a_large_pool():
    """Offsets beyond 32 bits, in elements, of one pool that holds keys and values interleaved."""
    import torch
    d, page, n_pages = 128, 64, 140000
    pool = torch.empty(n_pages, 2, 1, page, d, dtype=torch.float16, device="cuda")
    kp, vp = pool[:, 0], pool[:, 1]
    assert (n_pages - 1) * pool.stride(0) > 2 ** 31
    gen = torch.Generator(device="cuda").manual_seed(1)
    P = V.PagedKV(kp, vp, 4, torch.float32, rope_dim=0)
    n = 200
    table = torch.tensor([[n_pages - 1, 0, n_pages - 70, 139000]], dtype=torch.int32).cuda()
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    slots = table[0].long()[pos // page] * page + pos % page
    k, v = (torch.randn(n, d, generator=gen, device="cuda") for _ in range(2))
    q = torch.randn(n, 4 * d, generator=gen, device="cuda")
    means = torch.zeros(n_pages, 1, d, dtype=torch.float16, device="cuda")
    P.append(q, k, v, pos, slots, torch.empty_like(q), means=means)
    kv_len = torch.tensor([n], dtype=torch.int32).cuda()
    out = torch.empty(1, 4 * d, device="cuda")
    P.attn(q[:1], table, kv_len, out)
    P.sync()
    kk, vv = k.half().double()[None], v.half().double()[None]
    ref, s = plain_attn(q[0].double().reshape(1, 4, d), kk, vv, 1 / math.sqrt(d))
    assert ((out.double().reshape(1, 4, d) - ref).abs() <= attn_tol(ref, s, float(v.abs().max()), n, d, F32, F16)).all()
    m = means[table[0].long()[:3], 0].double()
    ref = kk[0, :192].reshape(3, 64, d).mean(1)
    assert ((m - ref).abs() <= 2.0 ** -11 * ref.abs() + 64 * STEP * 4 + 2.0 ** -24).all()
    del pool, kp, vp, P
    torch.cuda.empty_cache()


@gpu
def test_many_requests_and_long_lines():
    """More requests than a CTA has threads, and tables so wide that the line
    of tiles passes 32 bits."""
    import torch
    r = random.Random(4)
    lens = [r.choice([0, 1, 7, 64, 65, 300]) for _ in range(1100)]
    kp, vp, table, kv_len, q = make_requests(lens, 4, 2, 128, BF16, BF16, 16, False, 12)
    P = V.PagedKV(kp, vp, 4)
    out = torch.full_like(q, math.nan)
    P.attn(q, table, kv_len, out)
    P.sync()
    check_attn(out, q, kp, vp, table, lens, 4, BF16, BF16, 1 / math.sqrt(128), 16)
    wide = torch.full((1100, 200), -1, dtype=torch.int32, device="cuda")  # too wide for a CTA per pair
    wide[:, :table.shape[1]] = table
    out.fill_(math.nan)
    P.attn(q, wide, kv_len, out)
    P.sync()
    check_attn(out, q, kp, vp, table, lens, 4, BF16, BF16, 1 / math.sqrt(128), 16)
    lens = [1500, 0, 3, 900, 64, 1, 2000, 777]
    kp, vp, table, kv_len, q = make_requests(lens, 16, 16, 128, F32, F16, 1024, False, 13)
    P = V.PagedKV(kp, vp, 16, torch.float32)
    wide = torch.full((8, (1 << 21) - 1), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    out, narrow = torch.full_like(q, math.nan), torch.empty_like(q)
    P.attn(q, wide, kv_len, out)
    P.attn(q, table, kv_len, narrow)
    P.sync()
    check_attn(out, q, kp, vp, table, lens, 16, F32, F16, 1 / math.sqrt(128), 1024)
    assert torch.equal(out, narrow)
    del wide
    torch.cuda.empty_cache()


@gpu
def test_nothing_to_do():
    import torch
    kp, vp = (torch.zeros(2, 1, 8, 64, device="cuda") for _ in range(2))
    P = V.PagedKV(kp, vp, 2)
    z = lambda *s, d=torch.float32: torch.zeros(s, dtype=d, device="cuda")
    P.append(z(0, 128), z(0, 64), z(0, 64), z(0, d=torch.int32), z(0, d=torch.int64), z(0, 128))
    P.attn(z(0, 128), z(0, 3, d=torch.int32), z(0, d=torch.int32), z(0, 128))
    P.attn_topk(z(0, 128), z(0, 3, d=torch.int32), z(0, d=torch.int32), z(2, 1, 64), 0, 1, 1, z(0, 128))
    P.sync()
    with pytest.raises(V.VireoError):
        P.attn(z(1, 128), z(1, 3, d=torch.int64), z(1, d=torch.int32), z(1, 128))
    with pytest.raises(V.VireoError):
        P.attn(z(1, 64), z(1, 3, d=torch.int32), z(1, d=torch.int32), z(1, 128))
    with pytest.raises(V.VireoError):
        P.attn(z(1, 129)[:, 1:], z(1, 3, d=torch.int32), z(1, d=torch.int32), z(1, 128))  # 4-byte aligned
    with pytest.raises(V.VireoError):
        P.append(z(1, 128), z(1, 64), z(1, 64).half(), z(1, d=torch.int32), z(1, d=torch.int64), z(1, 128))
    with pytest.raises(V.VireoError):
        P.append(z(1, 128), z(1, 64), z(1, 64), z(1, d=torch.int32), z(1, d=torch.int64), z(1, 128), q_norm=z(65))
    x = z(3, 160)
    with pytest.raises(V.VireoError):  # in place, with another stride
        V.check(V.lib().gguf_kv_append(P.h, C.byref(V.GgufKvAppendArgs(
            3, x.data_ptr(), x.data_ptr(), x.data_ptr(), 160, 160, 160, x.data_ptr(), 144,
            z(3, d=torch.int32).data_ptr(), z(3, d=torch.int64).data_ptr())), None), "append")


@gpu
def test_streams_and_graphs():
    """On a side stream, by raw handle, captured, replayed on new inputs, and
    two captured graphs at once."""
    import torch
    lens = [500, 33, 0, 2100]
    args = (8, 2, 128, BF16, BF16, 16, False)
    kp, vp, table, kv_len, q = make_requests(lens, *args, 6)
    P = V.PagedKV(kp, vp, 8)
    means = torch.where(kp.isnan(), 0, kp).float().mean(2).to(kp.dtype).contiguous()
    want, want_k = torch.empty_like(q), torch.empty_like(q)
    P.attn(q, table, kv_len, want)
    P.attn_topk(q, table, kv_len, means, 1, 2, 9, want_k)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    a, b = torch.zeros_like(q), torch.zeros_like(q)
    with torch.cuda.stream(side):
        P.attn(q, table, kv_len, a)
        P.attn_topk(q, table, kv_len, means, 1, 2, 9, b)
    side.synchronize()
    assert torch.equal(a, want) and torch.equal(b, want_k)
    a.zero_()
    b.zero_()
    torch.cuda.synchronize()
    P.attn(q, table, kv_len, a, stream=side.cuda_stream)
    P.attn_topk(q, table, kv_len, means, 1, 2, 9, b, stream=side)
    P.sync(side)
    assert torch.equal(a, want) and torch.equal(b, want_k)
    graphs, outs = [], []
    for i in range(2):
        o = (torch.zeros_like(q), torch.zeros_like(q))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            P.attn(q, table, kv_len, o[0])
            P.attn_topk(q, table, kv_len, means, 1, 2, 9, o[1])
        graphs.append(g)
        outs.append(o)
    s2 = torch.cuda.Stream()
    for rep in range(20):
        for g, s in zip(graphs, (side, s2)):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o[0], want) and torch.equal(o[1], want_k)
    # new inputs in place: shorter and longer requests, another query
    q.copy_(torch.randn_like(q.float()).to(q.dtype))
    kv_len.copy_(torch.tensor([499, 0, 0, 1700], dtype=torch.int32))
    P.attn(q, table, kv_len, want)
    P.attn_topk(q, table, kv_len, means, 1, 2, 9, want_k)
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0][0], want) and torch.equal(outs[0][1], want_k)
    del graphs


@gpu
@pytest.mark.parametrize("act,kv,page,size", [(F32, F16, 16, 128), (BF16, BF16, 8, 64)])
def test_a_run_of_steps(act, kv, page, size):
    """Requests come, grow, end and give their pages to others: plan, append,
    attention and block attention step by step, the decode steps through one
    captured graph on a padded batch, against plain per-request caches."""
    import torch
    h, g, n_seq, width, rope_base, eps = 4, 2, 6, 12, 1e4, 1e-6
    n_pages, d, cap = 14, size, 64
    gen = torch.Generator(device="cuda").manual_seed(3)
    kp, vp = (make_pool(n_pages, g, page, d, dt(kv), False, gen, math.nan) for _ in range(2))
    P = V.PagedKV(kp, vp, h, dt(act), eps=eps, rope_base=rope_base)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
    table = torch.full((n_seq, width), -1, dtype=torch.int32, device="cuda")
    kv_len, add, granted, cu = i32([0] * n_seq), i32([0] * n_seq), i32([0] * n_seq), i32([0] * (n_seq + 1))
    ring, state = i32(list(range(n_pages))), i32([0, n_pages])
    slots, pos = torch.zeros(cap, dtype=torch.int64).cuda(), i32([0] * cap)
    means = torch.full((n_pages, g, d), math.nan, device="cuda", dtype=dt(kv))
    qn, kn = (torch.randn(d, generator=gen, device="cuda") * 0.1 + 1 for _ in range(2))
    qkv = torch.zeros(cap, (h + 2 * g) * d, device="cuda", dtype=dt(act))
    q_out = torch.zeros(cap, h * d, device="cuda", dtype=dt(act))
    out, out_k = (torch.zeros(n_seq, h * d, device="cuda", dtype=dt(act)) for _ in range(2))
    last = torch.zeros(n_seq, dtype=torch.int64).cuda()
    top = (1, 1, 2)

    def step():
        V.kv_plan(kv_len, add, table, ring, state, page, slots=slots, pos=pos, cu=cu, kv_len=kv_len, granted=granted,
                  state_out=state)
        P.append(qkv[:, :h * d], qkv[:, h * d:(h + g) * d], qkv[:, (h + g) * d:], pos, slots, q_out, q_norm=qn,
                 k_norm=kn, means=means)
        # a request's newest token
        torch.sub(cu[1:].long(), 1, out=last)
        qs = q_out[last.clamp(min=0)]
        P.attn(qs, table, kv_len, out)
        P.attn_topk(qs, table, kv_len, means, *top, out_k)
        return qs

    # warm-up of the graph on no tokens, then the capture
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qs = step()
    cache = [([], []) for _ in range(n_seq)]  # kept (key, value) rows as the pool must hold them
    pages = [[] for _ in range(n_seq)]
    rnd = random.Random(9)
    refused = 0
    for s in range(24):
        ask = []
        for i in range(n_seq):
            n = len(cache[i][0])
            ask.append(rnd.choice([3, 2 * page + 1]) if n == 0 else -1 if n > 4 * page or rnd.random() < 0.05 else 1)
        add.copy_(i32(ask))
        qkv.copy_(torch.randn(qkv.shape, generator=gen, device="cuda").to(qkv.dtype))
        q_out.fill_(math.nan)
        graph.replay()
        P.sync()
        ok, lens, start, ps, sl = granted.tolist(), kv_len.tolist(), cu.tolist(), pos.tolist(), slots.tolist()
        refused += ok.count(0)
        kk, kmag = plain_append_rows(qkv[:, h * d:(h + g) * d], None, kn, g, d, pos, d, rope_base, eps)
        vv = qkv[:, (h + g) * d:].double().reshape(cap, g, d)
        held = set()
        for i in range(n_seq):
            if ok[i] and ask[i] < 0:
                cache[i] = ([], [])
            for j in range(start[i], start[i + 1]):
                assert ps[j] == len(cache[i][0])
                assert sl[j] == table[i, ps[j] // page].item() * page + ps[j] % page
                cache[i][0].append(kk[j])
                cache[i][1].append(vv[j])
            n = len(cache[i][0])
            assert lens[i] == n
            mine = table[i, :-(-n // page)].tolist()
            assert not held & set(mine)
            held |= set(mine)
            if n == 0:
                assert (out[i] == 0).all() and (out_k[i] == 0).all()
                continue
            if start[i + 1] == start[i]:
                continue
            # the pool holds the rows, each rounded once
            k, v = rows_of(kp, table[i, :len(mine)], n), rows_of(vp, table[i, :len(mine)], n)
            rk, rv = torch.stack(cache[i][0], 1), torch.stack(cache[i][1], 1)
            assert ((k - rk).abs() <= 2 * half_eps(dt(kv)) * rk.abs() + 1e-4).all()
            assert ((v - rv).abs() <= half_eps(dt(kv)) * rv.abs() + 1e-7).all()
            sc = 1 / math.sqrt(d)
            ref, sm = plain_attn(qs[i].double().reshape(g, h // g, d), k, v, sc)
            err = (out[i].double().reshape(g, h // g, d) - ref).abs()
            assert (err <= attn_tol(ref, sm, float(v.abs().max()), n, d, act, kv)).all()
            for a in range(g):
                qa = qs[i].reshape(g, h // g, d)[a].double()
                ch = plain_select(qa.cpu().numpy(), means[table[i, :len(mine)].long(), a].double().cpu().numpy(), n,
                                  page, *top)
                at = torch.tensor([j for p in ch for j in range(p * page, min(n, (p + 1) * page))]).cuda()
                ref, sm = plain_attn(qa[None], k[a:a + 1, at], v[a:a + 1, at], sc)
                err = (out_k[i].double().reshape(g, h // g, d)[a] - ref[0]).abs()
                assert (err <= attn_tol(ref[0], sm, float(v.abs().max()), len(at), d, act, kv)).all()
        assert state.tolist()[1] == n_pages - len(held)
        live = start[-1]
        assert q_out[:live].isfinite().all() and q_out[live:].isnan().all()
    assert refused > 0  # the pool ran out at times
    del graph


# ---------------------------------------------------------------------------
# limits
# ---------------------------------------------------------------------------

_PLANS_IN_ORDER = """
import sys
import torch
sys.path[:0] = sys.argv[1:3]
import test_paged_kv as T
import vireo_b200 as V
for n in map(int, sys.argv[4:]):
    past, add, table, ring, state, n_slots = T.plan_case(n, 16, 6, n, 0)
    want = T.plain_plan(past, add, [r[:] for r in table], ring[:], state, 16, n_slots)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
    new = lambda k, d=torch.int32: torch.full((k,), 99, dtype=d, device="cuda")
    t, ri, pa, s = i32(table), i32(ring), i32(past), i32(state)
    slots, pos, cu, gr = new(n_slots, torch.int64), new(n_slots), new(n + 1), new(n)
    kv, so = (pa, s) if sys.argv[3] == "in place" else (new(n), new(2))
    V.kv_plan(pa, i32(add), t, ri, s, 16, slots=slots, pos=pos, cu=cu, kv_len=kv, granted=gr, state_out=so)
    got = [x.cpu().tolist() for x in (t, ri, slots, pos, cu, kv, gr, so)]
    assert got == list(want), n
print("all right")
"""


@gpu
@pytest.mark.parametrize("where", ["apart", "in place"])
def test_plan_of_as_many_requests_as_default_shared_memory_holds(where):
    """The request counts around 48 KB of lengths, in a process of their own
    and in rising order: no larger call has raised the kernel's limit before."""
    import os
    import subprocess
    import sys
    here = os.path.dirname(os.path.abspath(__file__))
    r = subprocess.run([sys.executable, "-c", _PLANS_IN_ORDER, here, os.path.dirname(here), where, "4010", "4011",
                        "4079", "4080", "4095", "4096"], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0 and "all right" in r.stdout, r.stdout + r.stderr


@gpu
def test_plan_of_asks_beyond_31_bits():
    """What is asked for in all passes 2^31 and more: nobody is granted on a
    sum that wrapped, with lengths and state apart and in place."""
    import torch
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
    big, page, width, n_pages = 2 ** 30, 1024, 2 ** 21 - 1, 8
    for adds in ([big, big, 5], [big, big, 5, big, big, 5], [big] * 7 + [5, 4, 0], [2 ** 31 - 1024] * 40 + [5, 0, -1]):
        n = len(adds)
        past = [0 if a >= big else 100 for a in adds]
        table = torch.full((n, width), -1, dtype=torch.int32, device="cuda")
        table[:, 0] = i32([-1 if a >= big else 7 for a in adds])
        for in_place in (False, True):
            p, s, ring = i32(past), i32([3, 7]), i32([5, 6, -2, 0, 1, 2, 3, 4])
            slots, pos = torch.full((4,), 9, dtype=torch.int64, device="cuda"), i32([9] * 4)
            cu, gr = i32([9] * (n + 1)), i32([9] * n)
            kv, so = (p, s) if in_place else (i32([9] * n), i32([9, 9]))
            V.kv_plan(p, i32(adds), table, ring, s, page, slots=slots, pos=pos, cu=cu, kv_len=kv, granted=gr,
                      state_out=so)
            ends = adds.count(-1)
            assert gr.tolist() == [int(a <= 0) for a in adds], adds
            assert kv.tolist() == [x if a >= 0 else 0 for x, a in zip(past, adds)]
            assert cu.tolist() == [0] * (n + 1) and slots.tolist() == [-1] * 4 and pos.tolist() == [0] * 4
            assert so.tolist() == [3, 7 + ends] and ring.tolist()[2] == (7 if ends else -2)
            assert (table[:, 1:8] == -1).all()
        del table
    torch.cuda.empty_cache()


@gpu
def test_plan_at_the_largest_number_of_slots():
    """n_slots = 2^30, the limit: asks of one token more than that are refused, asks of just that are granted."""
    import torch
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
    n_slots, page = 2 ** 30, 1024
    width = n_slots // page + 1
    n_pages = 2 * width + 3
    slots = torch.empty(n_slots, dtype=torch.int64, device="cuda")
    pos = torch.empty(n_slots, dtype=torch.int32, device="cuda")
    ids = torch.randperm(n_pages, device="cuda").to(torch.int32)
    half = n_slots // 2
    for adds, ok in (([half + 16, half + 16], [1, 0]), ([n_slots + 16], [0]), ([n_slots + 1, 1], [0, 0]),
                     ([n_slots], [1]), ([half, half], [1, 1]), ([half, half, 1, 0], [1, 1, 0, 1]),
                     ([n_slots, n_slots, 7], [1, 0, 0])):
        n = len(adds)
        table = torch.full((n, width), -1, dtype=torch.int32, device="cuda")
        cu, kv, gr, so = i32([9] * (n + 1)), i32([9] * n), i32([9] * n), i32([9, 9])
        slots.fill_(9)
        pos.fill_(9)
        V.kv_plan(i32([0] * n), i32(adds), table, ids, i32([n_pages - 5, n_pages]), page, slots=slots, pos=pos, cu=cu,
                  kv_len=kv, granted=gr, state_out=so)
        got = [a * g for a, g in zip(adds, ok)]
        assert gr.tolist() == ok and kv.tolist() == got, adds
        starts = [sum(got[:i]) for i in range(n + 1)]
        assert cu.tolist() == starts
        taken = 0
        for i, g in enumerate(got):
            need = -(-g // page)
            row = ids[(n_pages - 5 + taken + torch.arange(need, device="cuda")) % n_pages]
            assert torch.equal(table[i, :need], row) and (table[i, need:] == -1).all()
            taken += need
            for lo in range(0, g, 1 << 26):  # a part at a time
                j = torch.arange(lo, min(g, lo + (1 << 26)), device="cuda")
                at = slice(starts[i] + lo, starts[i] + lo + j.numel())
                assert torch.equal(pos[at], j.int()) and torch.equal(slots[at], row[j // page].long() * page + j % page)
        assert (slots[starts[-1]:] == -1).all() and (pos[starts[-1]:] == 0).all()
        assert so.tolist() == [(n_pages - 5 + taken) % n_pages, n_pages - taken]
    del slots, pos
    torch.cuda.empty_cache()


@gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("gap", [8.0, 11.0, 14.0, 17.5, 18.5, 20.0])
@pytest.mark.parametrize("act,kv", PAIRS)
def test_attn_beside_dominant_keys(act, kv, gap, d):
    """Keys that outweigh all others by e^gap, with values of zero: the rest,
    thousands of weights down to e^-gap and all of one sign, is the output.

    Requests share their pages, so that a stretch of thousands of positions
    stays in one CTA, and every warp has a dominant key.  Only dimension 0 of
    q and keys is not zero, q is 1 and the scale 1: a score s is a key's value
    exactly.  In steps of 2^-24, relative to the output: a weight's argument
    is off by 2.5 |s| + 2.5 |max| + |s - max| <= 8 S, one more of 14 and of
    its size, for the weight and for its share of the sum, hence twice; exp2
    4 and again twice; the split over two values 4 (bf16: 2^8); sums of
    positive terms, a step or two a tile and 64 for the joins."""
    import torch
    n, page, g, r, seqs = 8189, 16, 8, 2, 64
    gen = torch.Generator(device="cuda").manual_seed(17)
    need = -(-n // page)
    kp, vp = (torch.zeros(need, g, page, d, dtype=dt(kv), device="cuda") for _ in range(2))
    score = torch.randn(need * page, generator=gen, device="cuda") * 0.5
    score[:128] = gap
    kp[..., 0] = score.view(need, 1, page).to(dt(kv))
    vp.copy_((torch.rand(need, g, page, d, generator=gen, device="cuda") + 0.5).to(dt(kv)))
    vp[:128 // page] = 0
    table = torch.randperm(need, generator=gen, device="cuda").to(torch.int32)
    kp, vp = (torch.empty_like(x).index_copy_(0, table.long(), x) for x in (kp, vp))
    q = torch.zeros(seqs, g * r, d, dtype=dt(act), device="cuda")
    q[..., 0] = 1.0
    out = torch.full_like(q, math.nan)
    P = V.PagedKV(kp, vp, g * r, dt(act))
    P.attn(q, table.expand(seqs, need).contiguous(), torch.full((seqs,), n, dtype=torch.int32, device="cuda"), out,
           scale=1.0)
    P.sync()
    k, v = rows_of(kp, table, n), rows_of(vp, table, n)
    ref, _ = plain_attn(q[0].double().reshape(g, r, d), k, v, 1.0)
    s = float(k[..., 0].abs().max())
    steps = 2 * (8 * s + 14 + 2 * gap + 4) + {F32: 0, F16: 4, BF16: 256}[kv] + 4 * (n / 32 + 64)
    tol = half_eps(dt(act)) * ref + steps * STEP * ref + (2.0 ** -25 if act == F16 else 0.0)
    err = (out.double().reshape(seqs, g, r, d) - ref).abs()
    assert (err <= tol).all(), float((err / tol).max())


@gpu
@pytest.mark.parametrize("r", [1, 8, 12])
@pytest.mark.parametrize("kv", [F16, F32])
def test_attn_of_queries_of_any_size(kv, r):
    """fp32 queries as large and as small as fp32 holds, and rows whose
    elements lie far apart, over either cache.  Scores stay finite in fp32."""
    import torch
    n, d, page, scale = 200, 64, 16, 0.125
    kp, vp, table, kv_len, q = make_requests([n], r, 1, d, F32, kv, page, False, 23)
    order = torch.randperm(n, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    pages = table[0, :-(-n // page)]

    def set_keys(make):
        for j in range(n):
            kp[pages[j // page].item(), :, j % page] = make(j).to(kp.dtype)
    P = V.PagedKV(kp, vp, r, torch.float32)
    out = torch.empty_like(q)
    v = rows_of(vp, pages, n)[0]
    zero = torch.zeros(d, device="cuda")
    # the largest score takes it all: keys order / 256 in dimension 0
    ramp = [float(x) / 256 for x in order.tolist()]

    def one_hot(x):
        y = zero.clone()
        y[0] = x
        return y
    set_keys(lambda j: one_hot(ramp[j]))
    best = v[ramp.index(max(ramp))]
    for e in (20, 90, 110, 116, 120, 127):
        q.zero_()
        q.view(r, d)[:, 0] = 2.0 ** e
        P.attn(q, table, kv_len, out, scale=scale)
        assert (out.double().view(r, d) == best).all(), e
    # scores of next to nothing: the mean
    for e in (-30, -100, -126, -149):
        q.zero_()
        q.view(r, d)[:, 0] = 2.0 ** e
        P.attn(q, table, kv_len, out, scale=scale)
        ref = v.mean(0)
        assert ((out.double().view(r, d) - ref).abs() <= attn_tol(ref, 0.0, float(v.abs().max()), n, d, F32, kv)).all()
    # a small element of q against large keys, beside a large one against none
    wide = [(x - 0.5) * 2 * 60000 for x in ramp]

    def second(x):
        y = zero.clone()
        y[1] = x
        return y
    set_keys(lambda j: second(wide[j]))
    q.zero_()
    q.view(r, d)[:, 0] = 1.0
    q.view(r, d)[:, 1] = torch.linspace(1, 2, r, device="cuda") * 2.0 ** -18 * 1.3711
    P.attn(q, table, kv_len, out, scale=1.0)
    ref, s = plain_attn(q.double().view(1, r, d), rows_of(kp, pages, n), v[None], 1.0)
    tol = attn_tol(ref[0], s, float(v.abs().max()), n, d, F32, kv)
    err = (out.double().view(r, d) - ref[0]).abs()
    assert (err <= tol).all(), float((err / tol).max())
    # an infinite element makes every score -inf, whatever the others are
    set_keys(lambda j: torch.where(torch.arange(d, device="cuda") == 0, -1.0 - ramp[j], 1.0))
    q.fill_(1e5)
    q.view(r, d)[:, 0] = math.inf
    P.attn(q, table, kv_len, out, scale=scale)
    assert (out == 0).all()
    P.sync()


@pytest.mark.parametrize("scale", [2.5e38, -3.4e38, math.inf])
def test_attn_refuses_a_scale_that_overflows(scale):
    """Scores are multiplied by scale * log2(e): that has to be finite too."""
    L = V._kv_api()
    st, h = create(kv_desc())
    try:
        a = V.GgufKvAttnArgs(n_seqs=2, max_pages=8, q=4096, q_stride=512, out=4096, out_stride=512, table=4096,
                             table_stride=8, kv_len=4096, scale=scale, ws=4096, ws_bytes=1 << 62)
        assert L.gguf_kv_attn(h, C.byref(a), None) == -1
        assert L.gguf_kv_attn_topk(h, C.byref(a), C.byref(V.GgufKvSelectArgs(4096, 1, 1, 2, None)), None) == -1
    finally:
        L.gguf_kv_destroy(h)


COVER_CASES = [
    # lens, heads, kv heads, size, (act, kv), page, tokens_first
    ([8200], 32, 4, 128, (F32, F16), 64, False),
    ([8200, 3], 16, 16, 128, (F32, F32), 16, False),
    ([40001, 0, 5], 8, 2, 64, (F32, F16), 8, False),
    ([9001, 3000, 0, 129, 1], 28, 4, 64, (F16, F16), 8, True),
    ([7200, 777], 32, 4, 128, (BF16, BF16), 16, False),
    ([2049, 4100, 64], 12, 1, 256, (BF16, BF16), 32, False),
    ([5000, 1], 16, 1, 128, (F32, F32), 1024, True),
    ([6001], 24, 2, 128, (F16, F16), 32, False),
    ([(131 * i) % 3001 for i in range(70)], 8, 4, 64, (F32, F32), 16, False),
    ([(131 * i) % 1201 for i in range(150)], 16, 4, 128, (F32, F16), 16, True),
    ([300] * 9, 16, 16, 128, (F32, F16), 16, False),
]


@gpu
@pytest.mark.parametrize("case", COVER_CASES, ids=lambda c: str(c)[-60:])
def test_attn_takes_every_position_once(case):
    """All weights are equal (q is zero) and a value says in two dimensions
    where its position stands, j mod half the size and j div that, mod that
    again: what a dimension counts is exact, and one position too many or too
    few shows."""
    import torch
    lens, h, g, d, (act, kv), page, tf = case
    kp, vp, table, kv_len, q = make_requests(lens, h, g, d, act, kv, page, tf, 41)
    q.zero_()
    m = d // 2

    def marks(j):
        x = torch.zeros(j.numel(), d, device="cuda")
        x.scatter_(1, (j % m)[:, None], 1.0).scatter_(1, (m + j // m % m)[:, None], 1.0)
        return x
    for i, n in enumerate(lens):
        j = torch.arange(n, device="cuda")
        vp[table[i].long()[j // page], :, j % page] = marks(j)[:, None].to(vp.dtype)
    P = V.PagedKV(kp, vp, h, dt(act))
    out, out_k = torch.full_like(q, math.nan), torch.full_like(q, math.nan)
    P.attn(q, table, kv_len, out)
    sink, window, top = 1, 2, 60  # all scores alike: the first pages and the last
    means = torch.zeros(kp.shape[0], g, d, device="cuda", dtype=kp.dtype)
    P.attn_topk(q, table, kv_len, means, sink, window, top, out_k)
    P.sync()
    for i, n in enumerate(lens):
        j = torch.arange(n, device="cuda")
        total = -(-n // page)
        kept = (total <= sink + window + top) | (j // page < sink + top) | (j // page >= total - window)
        for got, j in ((out[i], j), (out_k[i], j[kept])):
            if n == 0:
                assert (got == 0).all()
                continue
            count = marks(j).double().sum(0)
            # one more or less, 1 / count, is above two tolerances
            assert float(count[:m].max()) * half_eps(dt(act)) < 0.5
            ref = count / j.numel()
            # 1 / n, the product with it, the result
            err = (got.double().view(h, d) - ref).abs()
            assert (err <= (half_eps(dt(act)) + 2 * STEP) * ref).all(), (i, n, float(err.max() * j.numel()))


@gpu
@pytest.mark.parametrize("kv", [F32, F16])
@pytest.mark.parametrize("lens,h,g,d,page", [([8200], 32, 4, 128, 64), ([1000, 300, 0, 17], 16, 16, 128, 16),
                                             ([2, 3, 1, 5000], 24, 2, 64, 8), ([900], 8, 1, 256, 32)])
def test_attn_errors_go_by_the_weights(lens, h, g, d, page, kv):
    """Small scores, fp32 outputs, and a bound that shrinks with a position's
    weight: leaving out or doubling one of thousands would break it.  Per
    value, in steps of sum p |v|: twice the score's (size + 4) S as above,
    exp2 and a weight's argument 12, its split 4, and the sums of both sides,
    a step a tile of a warp and 64 for the joins each."""
    import torch
    kp, vp, table, kv_len, q = make_requests(lens, h, g, d, F32, kv, page, False, 43, hot=0.3)
    P = V.PagedKV(kp, vp, h, torch.float32)
    out = torch.full_like(q, math.nan)
    P.attn(q, table, kv_len, out)
    P.sync()
    for i, n in enumerate(lens):
        if n == 0:
            continue
        pages, qs = table[i, :-(-n // page)], q[i].double().reshape(g, h // g, d)
        k, v = rows_of(kp, pages, n), rows_of(vp, pages, n)
        ref, s = plain_attn(qs, k, v, 1 / math.sqrt(d))
        pv, _ = plain_attn(qs, k, v.abs(), 1 / math.sqrt(d))
        tol = half_eps(torch.float32) * ref.abs() + pv * (2 * (d + 4) * s + 16 + 2 * (n / 32 + 64)) * STEP
        err = (out[i].double().reshape(g, -1, d) - ref).abs()
        assert (err <= tol).all(), (i, n, float((err / tol).max()))


@gpu
@pytest.mark.parametrize("r", [1, 7, 12])
@pytest.mark.parametrize("kv", [F32, F16])
def test_attn_keeps_the_digits_of_queries_and_weights(kv, r):
    """Few positions and one product to a score: what rounding q (24 bits) or
    the weights to the cache's type would lose is far above the bound."""
    import torch
    lens, d, page = [2, 3, 16, 41], 64, 8
    kp, vp, table, kv_len, q = make_requests(lens, r, 1, d, F32, kv, page, False, 47)
    first = torch.arange(d, device="cuda") == 0
    kp.copy_(torch.where(first, kp, torch.zeros_like(kp)))
    q.copy_(torch.where(first.repeat(r), 1 + torch.rand_like(q), torch.zeros_like(q)))
    P = V.PagedKV(kp, vp, r, torch.float32)
    out = torch.full_like(q, math.nan)
    P.attn(q, table, kv_len, out, scale=1.0)
    P.sync()
    for i, n in enumerate(lens):
        pages, qs = table[i, :-(-n // page)], q[i].double().reshape(1, r, d)
        k, v = rows_of(kp, pages, n), rows_of(vp, pages, n)
        ref, s = plain_attn(qs, k, v, 1.0)
        pv, _ = plain_attn(qs, k, v.abs(), 1.0)
        # a weight's argument 8 S + 14 and 2 S more of its size, exp2 4, for the weight and the sum; the split of q
        # 4 S and of the weight 4; the sums 64 each
        tol = half_eps(torch.float32) * ref.abs() + pv * (2 * (14 * s + 18) + 4 + 128) * STEP
        err = (out[i].double().reshape(1, r, d) - ref).abs()
        assert (err <= tol).all(), (i, n, float((err / tol).max()))


@gpu
@pytest.mark.parametrize("kv", [F16, BF16])
def test_attn_keeps_the_digits_of_equal_weights(kv):
    """64 positions with one weight, the furthest from its rounding to the
    type that a key can give, beside a heavier one with a value of zero."""
    import torch
    n, r, d, page = 65, 4, 128, 16
    kp, vp, table, kv_len, q = make_requests([n], r, 1, d, kv, kv, page, False, 53)
    x = -1 - 2 * torch.arange(1000, dtype=torch.float64) / 1000
    x = x.to(dt(kv)).double()
    w = x.exp()
    x = float(x[((w.to(dt(kv)).double() - w).abs() / w).argmax()])
    kp.copy_(torch.where(kp.isnan(), kp, torch.zeros_like(kp)))
    j = torch.arange(1, n, device="cuda")
    kp[table[0].long()[j // page], 0, j % page, 0] = x
    vp[table[0, 0].long(), 0, 0] = 0
    vp[table[0].long()[j // page], 0, j % page] = torch.linspace(1, 2, d, device="cuda").to(vp.dtype)
    q.zero_()
    q.view(r, d)[:, 0] = 1
    out = torch.full_like(q, math.nan)
    P = V.PagedKV(kp, vp, r)
    P.attn(q, table, kv_len, out, scale=1.0)
    P.sync()
    pages = table[0, :-(-n // page)]
    ref, s = plain_attn(q.double().view(1, r, d), rows_of(kp, pages, n), rows_of(vp, pages, n), 1.0)
    tol = half_eps(dt(kv)) * ref + (2 * (10 * s + 18) + {F16: 4, BF16: 256}[kv] + 128) * STEP * ref
    err = (out.double().view(1, r, d) - ref).abs()
    assert (err <= tol).all(), float((err / tol).max())


@gpu
def test_workspace_sizes_are_not_kept_for_ever():
    """Of thousands of different calls a pool remembers a few sizes."""
    import torch
    kp, vp = (torch.zeros(2, 1, 8, 64, device="cuda") for _ in range(2))
    P = V.PagedKV(kp, vp, 1)
    q = torch.zeros(1, 64, device="cuda")
    kv_len = torch.ones(1, dtype=torch.int32, device="cuda")
    table = torch.zeros(1, 3000, dtype=torch.int32, device="cuda")
    for width in range(1, 3001):
        P.attn(q, table[:, :width], kv_len, q)
    P.sync()
    held = sum(len(x) for x in vars(P).values() if isinstance(x, dict))
    assert held <= 1024, held


@gpu
def test_streams_by_every_name():
    """The default stream as an object, as 0 and by its own handle, the
    thread's default stream, and others: all run the call and give it memory."""
    import torch
    kp, vp, table, kv_len, q = make_requests([500, 33, 0, 2100], 8, 2, 128, BF16, BF16, 16, False, 6)
    P = V.PagedKV(kp, vp, 8)
    means = torch.where(kp.isnan(), 0, kp).float().mean(2).to(kp.dtype).contiguous()
    want, want_k = torch.empty_like(q), torch.empty_like(q)
    P.attn(q, table, kv_len, want)
    P.attn_topk(q, table, kv_len, means, 1, 2, 9, want_k)
    side = torch.cuda.Stream()
    for s in (torch.cuda.default_stream(), 0, 1, 2, side, side.cuda_stream, torch.cuda.ExternalStream(side.cuda_stream)):
        for inside in (torch.cuda.default_stream(), side):
            a, b = torch.zeros_like(q), torch.zeros_like(q)
            torch.cuda.synchronize()
            with torch.cuda.stream(inside):
                P.attn(q, table, kv_len, a, stream=s)
                P.attn_topk(q, table, kv_len, means, 1, 2, 9, b, stream=s)
                P.sync(s)
            torch.cuda.synchronize()
            assert torch.equal(a, want) and torch.equal(b, want_k), s


@gpu
@pytest.mark.parametrize("n,d", [(9000, 64), (65536, 128), (200001, 256)])
@pytest.mark.parametrize("act,kv", PAIRS)
def test_attn_sums_do_not_drift(act, kv, n, d):
    """Long sums of one sign that stay in one CTA (requests share their pages).
    Scores are 0, but for 128 first ones of 1.3 with values of zero, which
    make the other weights e^-1.3.  In steps of 2^-24 of the result: the
    weights as beside dominant keys; on tensor cores 2 for each product added
    to an accumulator, 32 at most, and one a run of 32 tiles (of 64 or more
    positions); on CUDA cores additions to nearest, four times the root of
    their number for each side; 64 for the joins."""
    import torch
    g, page, seqs, s = 8, 64, 96, 1.3
    gen = torch.Generator(device="cuda").manual_seed(19)
    need = -(-n // page)
    kp, vp = (torch.zeros(need, g, page, d, dtype=dt(kv), device="cuda") for _ in range(2))
    vp.copy_(torch.rand(vp.shape, generator=gen, device="cuda") + 0.5)
    table = torch.randperm(need, generator=gen, device="cuda").to(torch.int32)
    kp[table[:2].long(), :, :, 0], vp[table[:2].long()] = s, 0
    q = torch.zeros(seqs, g, d, dtype=dt(act), device="cuda")
    q[..., 0] = 1
    out = torch.full_like(q, math.nan)
    P = V.PagedKV(kp, vp, g, dt(act))
    P.attn(q, table.expand(seqs, need).contiguous(), torch.full((seqs,), n, dtype=torch.int32, device="cuda"), out,
           scale=1.0)
    P.sync()
    steps = 2 * (8 * s + 14 + 2 * s + 4) + {F32: 0, F16: 4, BF16: 256}[kv] + 64
    steps += 8 * math.sqrt(n) if kv == F32 else 64 + n / 1024
    top = math.exp(float(kp[table[0].long(), 0, 0, 0]))  # as the cache holds it
    for a in range(g):
        v = vp[:, a][table.long()].reshape(-1, d)[:n].double()
        ref = v.sum(0) / (n - 128 + 128 * top)
        tol = (half_eps(dt(act)) + steps * STEP) * ref
        err = (out[:, a].double() - ref).abs()
        assert (err <= tol).all(), (a, float((err / tol).max()))
