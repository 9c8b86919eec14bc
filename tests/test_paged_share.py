"""Requests that share pages of the key-value pool (gguf_kv_attn_shared,
gguf_kv_fork, gguf_kv_copy, gguf_kv_compact) and a beam search's choice
(gguf_beam_select), through the Python binding and, for refusals, the C-ABI,
against their definitions on lists or in 64 bits.

Tolerances: the attention's are those of gguf_kv_attn (test_paged_kv.py), from
the same arithmetic; a total of a beam's continuation is rounded once to fp32
(eps / 2 of its magnitude) after log sum exp that is off by at most 2^-19;
everything else is whole numbers or copies and is equal.
"""
import ctypes as C
import math
import random

import pytest

import vireo_b200 as V
from test_paged_kv import BF16, F16, F32, PAIRS, check_attn, create, dt, kv_desc, make_pool, plain_attn, attn_tol, \
    rows_of

gpu = pytest.mark.gpu


def i32(x):
    import torch
    return torch.tensor(x, dtype=torch.int32).cuda()


# ---------------------------------------------------------------------------
# refusals: host checks, no device needed
# ---------------------------------------------------------------------------

def test_packed_arguments_have_the_structures_layout():
    for pack, st in ((V._GROUP_PACK, V.GgufKvGroupArgs), (V._FORK_PACK, V.GgufKvForkArgs),
                     (V._COPY_PACK, V.GgufKvCopyArgs), (V._COMPACT_PACK, V.GgufKvCompactArgs),
                     (V._BEAM_PACK, V.GgufBeamArgs)):
        vals = [i + 1 for i, _ in enumerate(st._fields_)]
        raw = pack(*vals)
        assert len(raw) == C.sizeof(st)
        back = st.from_buffer_copy(raw)
        assert [getattr(back, n) for n, _ in st._fields_] == vals


SHARED_OK = dict(n_seqs=2, max_pages=8, q=4096, q_stride=512, out=4096, out_stride=512, table=4096, table_stride=8,
                 kv_len=4096, scale=0.0, ws=4096, ws_bytes=1 << 40)


@pytest.mark.parametrize("over,groups,status", [
    (dict(n_seqs=-1), (1, 4096, 4096), -1), (dict(max_pages=0), (1, 4096, 4096), -1),
    (dict(q=4104), (1, 4096, 4096), -1), (dict(out=None), (1, 4096, 4096), -1), (dict(ws=None), (1, 4096, 4096), -1),
    (dict(ws=4096 + 128), (1, 4096, 4096), -1), (dict(ws_bytes=1000), (1, 4096, 4096), -1),
    (dict(scale=float("inf")), (1, 4096, 4096), -1), (dict(out_stride=1024), (1, 4096, 4096), -1),
    (dict(table_stride=7), (1, 4096, 4096), -1),
    (dict(), (-1, 4096, 4096), -1), (dict(), (1, None, 4096), -1), (dict(), (1, 4096, None), -1),
    (dict(), (2 ** 20 + 1, 4096, 4096), -3), (dict(n_seqs=2 ** 17 + 1), (1, 4096, 4096), -3),
    (dict(), (8193, 4096, 4096), -3), (dict(n_seqs=8193), (1, 4096, 4096), -3),
    # a line of tiles that does not fit 32 bits
    (dict(n_seqs=8192, max_pages=2 ** 20, table_stride=2 ** 20), (1, 4096, 4096), -3)])
def test_attn_shared_refuses(over, groups, status):
    L = V._kv_api()
    st, h = create(kv_desc())
    try:
        f = dict(SHARED_OK)
        f.update(over)
        a, g = V.GgufKvAttnArgs(**f), V.GgufKvGroupArgs(*groups)
        assert L.gguf_kv_attn_shared(h, C.byref(a), C.byref(g), None) == status
    finally:
        L.gguf_kv_destroy(h)


def test_attn_shared_refuses_what_has_no_shape():
    L = V._kv_api()
    st, h = create(kv_desc())
    st2, wide = create(kv_desc(n_heads=130, n_kv_heads=1))
    try:
        a, g = V.GgufKvAttnArgs(**dict(SHARED_OK, q_stride=130 * 64, out_stride=130 * 64)), V.GgufKvGroupArgs(1, 4096, 4096)
        assert L.gguf_kv_attn_shared(h, C.byref(a), None, None) == -1
        assert L.gguf_kv_attn_shared(h, None, C.byref(g), None) == -1
        assert L.gguf_kv_attn_shared(None, C.byref(a), C.byref(g), None) == -1
        assert L.gguf_kv_attn_shared(wide, C.byref(a), C.byref(g), None) == -3  # more heads to a kv head than a tile
        assert L.gguf_kv_shared_workspace(None, 1, 1) == 0 and L.gguf_kv_shared_workspace(h, -1, 1) == 0
        assert L.gguf_kv_shared_workspace(h, 1, -1) == 0 and L.gguf_kv_shared_workspace(h, 2 ** 20, 1) == 0
        assert 0 < L.gguf_kv_shared_workspace(h, 4, 1) < L.gguf_kv_shared_workspace(h, 400, 1)
    finally:
        L.gguf_kv_destroy(h)
        L.gguf_kv_destroy(wide)


FORK_OK = dict(n_seqs=2, n_out=3, page_size=16, n_pages=9, max_pages=4, table_stride=4, table_out_stride=4,
               kv_len=4096, table=4096, parent=4096, keep=None, shares=4096, ring=4096, state=4096, table_out=8192,
               kv_len_out=8192, granted=4096, shares_out=4096, state_out=4096, src=4096, dst=4096, rows=4096, ws=4096,
               ws_bytes=1 << 20)


@pytest.mark.parametrize("over,status", [
    (dict(n_seqs=-1), -1), (dict(n_out=-1), -1), (dict(n_pages=0), -1), (dict(max_pages=0), -1),
    (dict(page_size=0), -1), (dict(page_size=24), -3), (dict(page_size=4), -3), (dict(n_seqs=8193), -3),
    (dict(n_out=8193), -3), (dict(max_pages=1 << 28, table_stride=1 << 28, table_out_stride=1 << 28), -1),
    (dict(table_stride=3), -1), (dict(table_out_stride=3), -1), (dict(kv_len=None), -1), (dict(table=None), -1),
    (dict(parent=None), -1), (dict(shares=None), -1), (dict(shares_out=None), -1), (dict(ring=None), -1),
    (dict(state=None), -1), (dict(state_out=None), -1), (dict(table_out=None), -1), (dict(table_out=4096), -1),
    (dict(kv_len_out=None), -1), (dict(granted=None), -1), (dict(src=None), -1), (dict(dst=None), -1),
    (dict(rows=None), -1), (dict(ws=None), -1), (dict(ws=4096 + 16), -1), (dict(ws_bytes=100), -1),
    (dict(kv_len_out=4096), -1), (dict(n_pages=2 ** 30 + 1), -3)])
def test_fork_refuses(over, status):
    f = dict(FORK_OK)
    f.update(over)
    L = V._kv_api()
    assert L.gguf_kv_fork(C.byref(V.GgufKvForkArgs(**f)), None) == status
    assert L.gguf_kv_fork(None, None) == -1
    assert L.gguf_kv_fork_workspace(8193, 1) == 0 and L.gguf_kv_fork_workspace(1, -1) == 0
    assert L.gguf_kv_fork_workspace(0, 0) > 0


COMPACT_OK = dict(n_seqs=2, page_size=16, n_pages=9, max_pages=4, n_copies=4, table_stride=4, table_out_stride=4,
                  kv_len=4096, table=4096, shares=4096, table_out=8192, shares_out=4096, ring=4096, state_out=4096,
                  src=4096, dst=4096, ws=4096, ws_bytes=1 << 20)


@pytest.mark.parametrize("over,status", [
    (dict(n_seqs=-1), -1), (dict(n_copies=-1), -1), (dict(n_pages=0), -1), (dict(max_pages=0), -1),
    (dict(page_size=48), -3), (dict(n_seqs=8193), -3), (dict(table_stride=3), -1), (dict(table_out_stride=3), -1),
    (dict(kv_len=None), -1), (dict(table=None), -1), (dict(table_out=None), -1), (dict(shares=None), -1),
    (dict(shares_out=None), -1), (dict(ring=None), -1), (dict(state_out=None), -1), (dict(src=None), -1),
    (dict(dst=None), -1), (dict(ws=None), -1), (dict(ws_bytes=10), -1), (dict(table_out=4096, table_out_stride=5), -1),
    (dict(max_pages=1 << 28, table_stride=1 << 28, table_out_stride=1 << 28), -1), (dict(n_pages=2 ** 30 + 1), -3)])
def test_compact_refuses(over, status):
    f = dict(COMPACT_OK)
    f.update(over)
    L = V._kv_api()
    assert L.gguf_kv_compact(C.byref(V.GgufKvCompactArgs(**f)), None) == status
    assert L.gguf_kv_compact(None, None) == -1 and L.gguf_kv_compact_workspace(0) == 0


@pytest.mark.parametrize("other", [
    dict(n_kv_heads=1, page_stride=16 * 64), dict(head_size=128, head_stride=2048, page_stride=4096, pos_stride=128),
    dict(page_size=32, head_stride=32 * 64, page_stride=2 * 32 * 64), dict(n_pages=5), dict(kv_type=0),
    dict(page_stride=4096), dict(pos_stride=128, head_stride=64)])
def test_copy_refuses_pools_that_differ(other):
    L = V._kv_api()
    (_, a), (st, b) = create(kv_desc()), create(kv_desc(**other))
    assert st == 0
    try:
        hs = (C.c_void_p * 2)(a, b)
        assert L.gguf_kv_copy(C.byref(V.GgufKvCopyArgs(0, 2, C.addressof(hs), None, 4096, 4096, None)), None) == -1
    finally:
        L.gguf_kv_destroy(a)
        L.gguf_kv_destroy(b)


def test_copy_refuses():
    L = V._kv_api()
    _, a = create(kv_desc())
    try:
        hs, none, odd = (C.c_void_p * 1)(a), (C.c_void_p * 1)(None), (C.c_void_p * 1)(4104)
        at = C.addressof
        for args in ((-1, 1, at(hs), None, 4096, 4096, None), (1, -1, at(hs), None, 4096, 4096, None),
                     (1, 1, None, None, 4096, 4096, None), (1, 1, at(none), None, 4096, 4096, None),
                     (1, 1, at(hs), None, None, 4096, None), (1, 1, at(hs), None, 4096, None, None),
                     (1, 1, at(hs), at(odd), 4096, 4096, None)):
            assert L.gguf_kv_copy(C.byref(V.GgufKvCopyArgs(*args)), None) == -1
        assert L.gguf_kv_copy(C.byref(V.GgufKvCopyArgs(2 ** 30 + 1, 1, at(hs), None, 4096, 4096, None)), None) == -3
        assert L.gguf_kv_copy(None, None) == -1
        assert L.gguf_kv_copy(C.byref(V.GgufKvCopyArgs(0, 1, at(hs), None, None, None, None)), None) == 0
        assert L.gguf_kv_copy(C.byref(V.GgufKvCopyArgs(1, 0, None, None, 4096, 4096, None)), None) == 0
    finally:
        L.gguf_kv_destroy(a)


BEAM_OK = dict(n_seqs=2, n_beams=3, n_out=4, vocab=100, type=0, end_token=-1, logits=4096, stride=100, score=4096,
               done=None, score_out=4096, token=4096, parent=4096, done_out=None, ws=4096, ws_bytes=1 << 20)


@pytest.mark.parametrize("over,status", [
    (dict(n_seqs=-1), -1), (dict(n_beams=0), -1), (dict(n_out=0), -1), (dict(vocab=0), -1),
    (dict(vocab=1, stride=1), -1), (dict(end_token=100), -1), (dict(end_token=-2), -1), (dict(done=4096), -1),
    (dict(n_beams=33), -3), (dict(n_out=33), -3), (dict(vocab=2 ** 20 + 1, stride=2 ** 21), -3), (dict(type=8), -3),
    (dict(logits=None), -1), (dict(logits=4098), -1), (dict(stride=99), -1), (dict(score=None), -1),
    (dict(score_out=None), -1), (dict(token=None), -1), (dict(parent=None), -1), (dict(ws=None), -1),
    (dict(ws=4096 + 64), -1), (dict(ws_bytes=64), -1)])
def test_beam_select_refuses(over, status):
    f = dict(BEAM_OK)
    f.update(over)
    L = V._kv_api()
    assert L.gguf_beam_select(C.byref(V.GgufBeamArgs(**f)), None) == status
    assert L.gguf_beam_select(None, None) == -1
    assert L.gguf_beam_select(C.byref(V.GgufBeamArgs(**dict(BEAM_OK, n_seqs=0, logits=None))), None) == 0
    assert L.gguf_beam_workspace(1, 33, 1, 10) == 0 and L.gguf_beam_workspace(1, 1, 1, 10) > 0


def test_binding_refuses_host_tensors_and_other_shapes():
    import torch
    z, f = torch.zeros(4, dtype=torch.int32), torch.zeros(4)
    t = z.view(4, 1)
    with pytest.raises(V.VireoError):
        V.kv_fork(z, t, z, z, z, z[:2], 16, table_out=t, kv_len_out=z, granted=z, shares_out=z, state_out=z[:2],
                  src=z, dst=z, rows=z)
    with pytest.raises(V.VireoError):
        V.kv_compact(z, t, z, 16, table_out=t, state_out=z[:2], src=z, dst=z)
    with pytest.raises(V.VireoError):
        V.beam_select(f.view(4, 1), f, 1, score_out=f.view(4, 1), token=t, parent=t)
    V.kv_copy([], z, z)  # no layers: nothing to do


# ---------------------------------------------------------------------------
# rows that continue other rows
# ---------------------------------------------------------------------------

def plain_fork(kv_len, table, parent, keep, shares, ring, state, page, out):
    """gguf_kv_fork's definition, row by row, on lists (out and ring are changed)."""
    n_pages, (head, count) = len(ring), state
    width = len((table or out)[0]) if table or out else 0
    inside = lambda p: 0 <= p < n_pages
    had = [min(max(n, 0), width * page) for n in kv_len]
    want = [0 if p < 0 else had[p] if keep is None or keep[i] < 0 else min(keep[i], had[p])
            for i, p in enumerate(parent)]
    holders, children = list(shares), {}
    for i, p in enumerate(parent):
        children.setdefault(p, []).append(i)
    for i, n in enumerate(had):
        for p in table[i][:-(-n // page)]:
            if inside(p):
                holders[p] -= 1
    lens, granted, copies, used = [], [], [], 0
    for i, p in enumerate(parent):
        copy, ok = (-1, -1, 0), 1
        if p >= 0:
            whole, tail = divmod(want[i], page)
            row = table[p][:whole]
            if tail:
                last = table[p][whole]
                near = [j for j in children[p] if want[j] > whole * page]
                if (not inside(last) or shares[last] == 0) and near[0] == i and all(
                        want[j] < (whole + 1) * page for j in near):
                    row = row + [last]
                elif used < count:
                    copy = (last, ring[(head + used) % n_pages], tail)
                    used += 1
                else:
                    ok = 0
            if ok:
                for q in row:
                    if inside(q):
                        holders[q] += 1
                row = row + ([copy[1]] if tail and copy[2] else [])
                out[i][:len(row)] = row
        lens.append(want[i] if ok else 0)
        granted.append(ok)
        copies.append(copy)
    gone = [q for q in range(n_pages) if holders[q] < 0][:n_pages - count]
    for j, q in enumerate(gone):
        ring[(head + count + j) % n_pages] = q
    return (out, lens, granted, [max(h, 0) for h in holders], ring, [(head + used) % n_pages, count - used + len(gone)],
            [c[0] for c in copies], [c[1] for c in copies], [c[2] for c in copies])


def fork_case(n, m, page, width, seed, few=False):
    """Rows of which some already share pages, and children of all kinds."""
    r = random.Random(seed)
    kv_len, table = [], []
    ids = list(range(n * width + 3))
    r.shuffle(ids)
    shares = [0] * len(ids)
    for i in range(n):
        k = min(width * page, r.choice([0, 1, page - 1, page, page + 1, 2 * page, r.randrange(width * page + 1)]))
        row, pages = [-7] * width, -(-k // page)
        both = 0
        if i and r.random() < 0.4:  # begins with whole pages of the row before
            both = min(k, kv_len[i - 1]) // page
            both = r.randrange(both + 1)
            row[:both] = table[i - 1][:both]
            for p in row[:both]:
                shares[p] += 1
        for j in range(both, pages):
            row[j] = ids.pop()
        kv_len.append(k)
        table.append(row)
    parent = [r.choice([-1, r.randrange(n), r.randrange(n), min(i, n - 1)]) if n else -1 for i in range(m)]
    if m > 3 and n:
        parent[1] = parent[2] = parent[0]
    keep = [r.choice([-1, -1, r.randrange(width * page + 5), kv_len[p] if p >= 0 else 3,
                      kv_len[p] // page * page if p >= 0 else 0]) for p in parent]
    n_pages = len(shares)
    head = r.randrange(n_pages)
    free = ids[:2] if few else ids
    ring = [-3] * n_pages
    for j, p in enumerate(free):
        ring[(head + j) % n_pages] = p
    return kv_len, table, parent, keep, shares, ring, [head, len(free)]


def run_fork(kv_len, table, parent, keep, shares, ring, state, page, width, in_place=False, times=2):
    import torch
    n, m, n_pages = len(kv_len), len(parent), len(ring)
    wide = torch.full((m, width + 3), -9, dtype=torch.int32, device="cuda")
    t = i32(table).view(n, width)
    out, sh, st, ri = wide[:, :width], i32(shares), i32(state), i32(ring)
    new = lambda k: torch.full((k,), 99, dtype=torch.int32, device="cuda")
    lens, gr, src, dst, rows = new(m), new(m), new(m), new(m), new(m)
    so, ss = (sh, st) if in_place else (new(n_pages), new(2))
    for _ in range(1 if in_place else times):
        V.kv_fork(i32(kv_len), t, i32(parent), sh, ri, st, page, keep=None if keep is None else i32(keep),
                  table_out=out, kv_len_out=lens, granted=gr, shares_out=so, state_out=ss, src=src, dst=dst, rows=rows)
    assert (wide[:, width:] == -9).all()
    return [x.cpu().tolist() for x in (out, lens, gr, so, ri, ss, src, dst, rows)]


FORK_NAMES = ("table", "kv_len", "granted", "shares", "ring", "state", "src", "dst", "rows")


@gpu
@pytest.mark.parametrize("n,m,page,width,few", [
    (1, 1, 16, 3, False), (4, 4, 8, 5, False), (4, 9, 16, 5, True), (7, 3, 1024, 2, False), (64, 64, 16, 40, False),
    (64, 70, 8, 129, True), (513, 520, 32, 9, False), (3, 0, 16, 4, False), (0, 3, 16, 4, False),
    (1000, 1500, 8, 70, False), (8192, 8192, 16, 3, False)])
@pytest.mark.parametrize("cut", [False, True])
def test_fork_matches_the_definition(n, m, page, width, few, cut):
    kv_len, table, parent, keep, shares, ring, state = fork_case(n, m, page, width, 31 * n + m, few)
    keep = keep if cut else None
    for in_place in (False, True):
        got = run_fork(kv_len, table, parent, keep, shares, ring, state, page, width, in_place)
        want = plain_fork(kv_len, table, parent, keep, shares, list(ring), state, page, [[-9] * width for _ in parent])
        for name, a, b in zip(FORK_NAMES, got, want):
            assert a == b, (name, in_place)
    V.sync()  # nothing to report


@gpu
def test_fork_of_a_wide_table_and_a_large_pool():
    """Launch by launch instead of in one cluster: long rows, many pages."""
    page, width, n_pages = 8, 30000, 300000
    r = random.Random(3)
    ids = list(range(n_pages))
    r.shuffle(ids)
    kv_len = [width * page, width * page - 3, 17, 9 * page]
    table, shares = [], [0] * n_pages
    for k in kv_len:
        table.append([ids.pop() for _ in range(-(-k // page))])
        table[-1] += [-7] * (width - len(table[-1]))
    table[3][:9] = table[0][:9]
    for p in table[3][:9]:
        shares[p] += 1
    ring, state = [-3] * n_pages, [n_pages - 5, 50]
    for j in range(50):
        ring[(n_pages - 5 + j) % n_pages] = ids[j]
    parent, keep = [1, 1, 0, 2, -1, 3], [-1, -1, 70001, 12, -1, 72]
    for in_place in (False, True):
        got = run_fork(kv_len, table, parent, keep, shares, ring, state, page, width, in_place)
        want = plain_fork(kv_len, table, parent, keep, shares, list(ring), state, page, [[-9] * width for _ in parent])
        for name, a, b in zip(FORK_NAMES, got, want):
            assert a == b, (name, in_place)


@gpu
def test_fork_reports_what_does_not_fit():
    """Parents that are no rows, lengths beyond the table, page numbers outside
    the pool, a page in two rows that counts one holder."""
    page, width, n_pages = 16, 3, 12
    base = dict(kv_len=[48, 20], table=[[0, 1, 2], [3, 4, -7]], parent=[0, 1], keep=None, shares=[0] * n_pages,
                ring=[5, 6, 7] + [-3] * 9, state=[0, 3])
    for over, same in ((dict(parent=[2, 1]), dict(parent=[-1, 1])), (dict(parent=[-5, 1]), dict(parent=[-1, 1])),
                       (dict(kv_len=[49, 20]), {}), (dict(kv_len=[48, -4]), dict(kv_len=[48, 0])),
                       (dict(table=[[0, -1, 2], [3, n_pages, -7]], parent=[0, 0]), None),
                       (dict(table=[[0, 1, 2], [0, 4, -7]], parent=[-1, -1]), None)):
        c = dict(base)
        c.update(over)
        got = run_fork(**c, page=page, width=width, times=1)
        if over != dict(kv_len=[48, -4]):
            with pytest.raises(V.VireoError) as e:
                V.sync()
            assert e.value.status == -1
        c.update(same or {})
        c["ring"] = list(c["ring"])
        c["parent"] = [p if 0 <= p < 2 else -1 for p in c["parent"]]
        want = plain_fork(**c, page=page, out=[[-9] * width for _ in c["parent"]])
        for name, a, b in zip(FORK_NAMES, got, want):
            assert a == b, (name, over)
    V.sync()


# ---------------------------------------------------------------------------
# copies
# ---------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("g,page,d,kv,tf", [(2, 16, 64, F16, False), (4, 64, 128, BF16, True), (1, 8, 64, F32, False),
                                            (3, 8, 128, F16, True), (5, 1024, 64, BF16, False),
                                            (2, 32, 256, F32, True)])
@pytest.mark.parametrize("layers", [1, 3])
def test_copy(g, page, d, kv, tf, layers):
    import torch
    gen = torch.Generator(device="cuda").manual_seed(g * page + layers)
    n_pages, r = 40, random.Random(page)
    pools = [[make_pool(n_pages, g, page, d, dt(kv), tf, gen, None) for _ in range(2)] for _ in range(layers)]
    means = [torch.randn(n_pages, g, d, generator=gen, device="cuda").to(dt(kv)) if i != 1 else None
             for i in range(layers)]
    handles = [V.PagedKV(k, v, g) for k, v in pools]
    ids = list(range(n_pages))
    r.shuffle(ids)
    src, dst, rows = ids[:12], ids[12:24], [r.choice([0, 1, page - 1, page, page + 9]) for _ in range(12)]
    src[3], dst[4], rows[5] = -1, src[4], -2
    src[7] = src[6]  # one page to two
    for count, with_means in ((rows, False), (None, True), (rows, True)):
        before = [[p.clone() for p in pair] for pair in pools]
        kept = [m.clone() if m is not None else None for m in means]
        V.kv_copy(handles if layers > 1 else handles[0], i32(src), i32(dst), rows=None if count is None else i32(count),
                  means=(means if layers > 1 else means[0]) if with_means else None)
        handles[0].sync()
        for pair, old in zip(pools, before):
            for p, want in zip(pair, old):
                for i, (a, b) in enumerate(zip(src, dst)):
                    k = page if count is None else min(max(count[i], 0), page)
                    if a >= 0:
                        want[b, :, :k] = want[a, :, :k].clone()
                assert torch.equal(p, want)
        for m, want in zip(means, kept):
            if m is not None:
                if with_means:
                    for a, b in zip(src, dst):
                        if a >= 0:
                            want[b] = want[a].clone()
                assert torch.equal(m, want)


@gpu
def test_copy_of_many_layers_and_of_pages_outside_the_pool():
    import torch
    layers, n_pages = 70, 6
    pool = torch.arange(layers * 2 * n_pages, device="cuda").float()[:, None].expand(-1, 8 * 64).reshape(
        layers, 2, n_pages, 1, 8, 64).contiguous()
    want = pool.clone()
    want[:, :, 4] = want[:, :, 1]
    handles = [V.PagedKV(pool[i, 0], pool[i, 1], 1) for i in range(layers)]
    V.kv_copy(handles, i32([6, 1, 2, -1, 3]), i32([0, 4, -1, 5, 6]))
    with pytest.raises(V.VireoError) as e:
        handles[0].sync()
    assert e.value.status == -1
    assert torch.equal(pool, want)
    handles[0].sync()  # reported once


# ---------------------------------------------------------------------------
# compaction
# ---------------------------------------------------------------------------

def plain_compact(kv_len, table, shares, n_pages, page, n_copies, out, ring):
    """gguf_kv_compact's definition, page by page, on lists."""
    width = len(out[0]) if out else 0
    have = [-(-min(max(n, 0), width * page) // page) for n in kv_len]
    used = {p for row, k in zip(table, have) for p in row[:k] if 0 <= p < n_pages}
    late = sorted(p for p in used if p >= len(used))
    src = late[max(0, len(late) - n_copies):]
    dst = [p for p in range(n_pages) if p not in used][:len(src)]
    to = dict(zip(src, dst))
    for row, o, k in zip(table, out, have):
        o[:k] = [to.get(p, p) for p in row[:k]]
    moved = list(shares)
    for a, b in to.items():
        moved[a], moved[b] = 0, shares[a]
    after = {to.get(p, p) for p in used}
    free = [p for p in range(n_pages) if p not in after]
    pad = [-1] * (n_copies - len(src))
    return out, moved, free + ring[len(free):], [0, len(free)], src + pad, dst + pad


@gpu
@pytest.mark.parametrize("n,page,width,n_pages,n_copies", [
    (1, 16, 3, 9, 4), (0, 16, 3, 5, 2), (6, 8, 7, 64, 64), (6, 8, 7, 64, 3), (6, 8, 7, 64, 0), (2, 16, 16, 32, 8),
    (300, 32, 20, 9001, 9001), (40, 8, 500, 40000, 777), (5, 8, 130, 1025, 99), (8192, 1024, 2, 20000, 5000),
    (8, 16, 8, 64, 10)])
def test_compact_matches_the_definition(n, page, width, n_pages, n_copies):
    import torch
    r = random.Random(n + n_pages)
    ids = list(range(n_pages))
    r.shuffle(ids)
    kv_len, table, shares = [], [], [0] * n_pages
    for i in range(n):
        most = min(width, max(1, 3 * n_pages // (4 * n)))
        k = r.choice([0, 1, page, most * page, r.randrange(most * page + 1)])
        if (n, n_pages) == (8, 64):
            k = width * page  # every page in use
        row = [ids.pop() for _ in range(-(-k // page))]
        if i and r.random() < 0.3:
            both = r.randrange(min(len(row), -(-kv_len[-1] // page)) + 1)
            ids += row[:both]
            row[:both] = table[-1][:both]
            for p in row[:both]:
                shares[p] += 1
        kv_len.append(k)
        table.append(row + [-7] * (width - len(row)))
    for in_place in (False, True):
        t, sh = i32(table).view(n, width), i32(shares)
        out = t if in_place else torch.full((n, width + 2), -9, dtype=torch.int32, device="cuda")[:, :width]
        so = sh if in_place else torch.full_like(sh, 99)
        ring, st, src, dst = i32([-3] * n_pages), i32([9, 9]), i32([8] * n_copies), i32([8] * n_copies)
        for _ in range(1 if in_place else 2):
            V.kv_compact(i32(kv_len), t, ring, page, shares=sh, table_out=out, shares_out=so, state_out=st, src=src,
                         dst=dst)
        got = [x.cpu().tolist() for x in (out, so, ring, st, src, dst)]
        fresh = [list(row) for row in table] if in_place else [[-9] * width for _ in table]
        want = plain_compact(kv_len, table, shares, n_pages, page, n_copies, fresh, [-3] * n_pages)
        for name, a, b in zip(("table", "shares", "ring", "state", "src", "dst"), got, want):
            assert a == b, (name, in_place)
    # without counts of holders
    t = i32(table).view(n, width)
    V.kv_compact(i32(kv_len), t, ring, page, table_out=t, state_out=st, src=src, dst=dst)
    assert t.cpu().tolist() == plain_compact(kv_len, table, shares, n_pages, page, n_copies,
                                             [list(row) for row in table], [-3] * n_pages)[0]
    V.sync()


@gpu
def test_compact_reports_what_does_not_fit():
    page, width, n_pages = 8, 3, 10
    kv_len, table = [24, 99], [[9, -1, 3], [n_pages, 8, 2 ** 31 - 1]]
    out, ring, st, src, dst = i32([[0] * 3] * 2), i32([0] * n_pages), i32([0, 0]), i32([0] * 4), i32([0] * 4)
    V.kv_compact(i32(kv_len), i32(table), ring, page, table_out=out, state_out=st, src=src, dst=dst)
    with pytest.raises(V.VireoError) as e:
        V.sync()
    assert e.value.status == -1
    want = plain_compact(kv_len, table, [0] * n_pages, n_pages, page, 4, [[0] * 3, [0] * 3], [0] * n_pages)
    assert [x.cpu().tolist() for x in (out, ring, st, src, dst)] == [want[0]] + list(want[2:])
    V.sync()


# ---------------------------------------------------------------------------
# the choice of a beam search
# ---------------------------------------------------------------------------

def plain_select(logits, score, beams, k, done, end):
    """gguf_beam_select's definition in 64 bits: per request [(total, row, token)], best first."""
    import torch
    out = []
    for s in range(0, logits.shape[0], beams):
        found = []
        for r in range(s, s + beams):
            sc = float(score[r])
            if not math.isfinite(sc):
                continue
            if done is not None and done[r]:
                found.append((sc, r, end))
                continue
            x = logits[r].double().cpu()
            lse = float(torch.logsumexp(x, 0))
            if not math.isfinite(lse):
                continue
            live = torch.nonzero(torch.isfinite(x))[:, 0]
            best = live[torch.argsort(x[live], descending=True, stable=True)][:k]
            found += [(sc + float(x[t]) - lse, r, int(t)) for t in best]
        found.sort(key=lambda f: (-f[0], f[1], f[2]))
        out.append(found[:k])
    return out


def check_select(logits, score, beams, k, done=None, end=-1):
    import torch
    n = logits.shape[0] // beams
    so = torch.full((n, k), 7.0, device="cuda")
    token, parent, dn = (torch.full((n, k), 99, dtype=torch.int32, device="cuda") for _ in range(3))
    for _ in range(2):
        V.beam_select(logits, score, beams, score_out=so, token=token, parent=parent, done=done, done_out=dn,
                      end_token=end)
    V.sync()
    want = plain_select(logits, score.cpu(), beams, k, None if done is None else done.cpu(), end)
    for i, found in enumerate(want):
        rest = k - len(found)
        assert token[i].tolist() == [f[2] for f in found] + [-1] * rest, i
        assert parent[i].tolist() == [f[1] for f in found] + [-1] * rest, i
        assert dn[i].tolist() == [int(f[2] == end) for f in found] + [1] * rest, i
        for got, f in zip(so[i].tolist(), found):
            assert abs(got - f[0]) <= 2.0 ** -24 * abs(f[0]) + 2.0 ** -19, (i, got, f)
        assert so[i, len(found):].tolist() == [-math.inf] * rest
    return so, token, parent


@gpu
@pytest.mark.parametrize("n,beams,k,vocab,t", [
    (1, 1, 1, 1, F32), (1, 1, 32, 32, F32), (3, 4, 4, 1000, F32), (2, 32, 32, 333, F16), (1, 3, 6, 50257, BF16),
    (5, 2, 7, 2049, F16), (9, 8, 8, 32001, F32), (2, 5, 1, 100003, BF16), (40, 8, 8, 9000, F32),
    (1, 32, 32, 300000, F32), (200, 2, 3, 17, F32)])
def test_beam_select(n, beams, k, vocab, t):
    import torch
    gen = torch.Generator(device="cuda").manual_seed(vocab)
    logits = (torch.randn(n * beams, vocab, generator=gen, device="cuda") * 3).to(dt(t))
    score = -torch.rand(n * beams, generator=gen, device="cuda") * 4 - 10
    check_select(logits, score, beams, k)
    # rows apart and at every alignment, some beams finished or unused
    done = (torch.rand(n * beams, generator=gen, device="cuda") < 0.3).int()
    score[torch.rand(n * beams, generator=gen, device="cuda") < 0.2] = -math.inf
    for stride, off in ((vocab + 1, 0), (vocab + 7, 3)):
        wide = torch.full((n * beams * stride + off,), math.nan, device="cuda").to(dt(t))
        view = wide[off:].view(n * beams, stride)[:, :vocab]
        view.copy_(logits)
        check_select(view, score, beams, k, done, vocab // 2)


@gpu
@pytest.mark.parametrize("vocab", [40, 5000, 40000])
def test_beam_select_ties_go_to_the_lower_index(vocab):
    """Rows of one value, rows of few values, rows that are the same, zeros of both signs."""
    import torch
    gen = torch.Generator(device="cuda").manual_seed(1)
    flat = torch.full((4, vocab), 1.5, device="cuda")
    zero = torch.zeros(4, device="cuda")
    check_select(flat, zero, 4, 11)
    few = torch.randint(0, 3, (6, vocab), generator=gen, device="cuda").float()
    few[1] = few[0]
    few[4] = few[0]
    check_select(few, zero.new_zeros(6), 3, 32)
    signed = torch.full((2, vocab), -5.0, device="cuda")
    signed[:, 3::4], signed[:, 1::4] = -0.0, 0.0
    check_select(signed, zero[:2], 2, 9)
    up = torch.arange(vocab, device="cuda").float()[None] / 64
    check_select(torch.cat([up, up.flip(1)]), zero[:2], 1, 32)


@gpu
@pytest.mark.parametrize("vocab", [50, 20000])
def test_beam_select_of_masked_infinite_and_nan_logits(vocab):
    import torch
    gen = torch.Generator(device="cuda").manual_seed(vocab)
    x = torch.randn(12, vocab, generator=gen, device="cuda")
    lowest = torch.finfo(torch.float32).min
    x[0] = -math.inf                      # nothing left
    x[1, 3:] = -math.inf                  # three tokens
    x[2, 7] = math.nan
    x[3, 8] = math.inf
    x[4] = lowest                         # the type's lowest everywhere
    x[5, :-2] = lowest
    x[7, 1:] = -math.inf
    score = torch.zeros(12, device="cuda")
    score[6], score[8], score[9] = -math.inf, math.nan, math.inf
    check_select(x, score, 6, 5)
    check_select(x, score, 1, 4)
    check_select(x, score, 4, 32, done=i32([1] * 12), end=0)  # four continuations at most
    check_select(x[:1], score[:1], 1, 3)                      # none


@gpu
@pytest.mark.parametrize("gap", [0.0, 1e-7, 4e-7, 1e-6, 3e-6])
def test_beam_select_tells_near_totals_of_two_rows_apart(gap):
    """The second row's score makes its best total lie a little above or below
    the first one's: by less than fp32 sums can tell, and in either direction."""
    import torch
    vocab, gen = 30000, torch.Generator(device="cuda").manual_seed(5)
    for sign in (1, -1):
        for seed in range(4):
            x = torch.randn(2, vocab, generator=gen, device="cuda") * 2
            lse = torch.logsumexp(x.double(), 1)
            top = x.max(1).values.double()
            # to fp32's step of a score, about 1e-7, and whichever way that falls
            want = float(top[0] - lse[0] - (top[1] - lse[1])) + sign * gap
            score = torch.tensor([0.0, want], dtype=torch.float64).float().cuda()
            check_select(x, score, 2, 6)


# ---------------------------------------------------------------------------
# attention over a shared prefix
# ---------------------------------------------------------------------------

def make_groups(groups, h, g, d, act, kv, page, tf, seed, hot=1.0):
    """groups: (shared positions, [own lengths]) or a bare own length.  A pool
    whose unused places hold NaN; cu and shared of the groups, which stand in
    one run (bare lengths before and behind them)."""
    import torch
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rows, lens, cu, shared = [], [], [], []
    fills, used = [], 0
    for e in groups:
        s, own = e if isinstance(e, tuple) else (0, [e])
        both = list(range(used, used + s // page))
        used += len(both)
        fills += [(p, page) for p in both]
        if isinstance(e, tuple):
            cu.append(len(lens))
            shared.append(s)
        for n in own:
            n = n + len(both) * page if n >= 0 else -n  # below zero: the length in all, less than what is shared
            extra = max(0, -(-n // page) - len(both))
            mine = list(range(used, used + extra))
            used += extra
            fills += [(p, min(page, n - (len(both) + j) * page)) for j, p in enumerate(mine)]
            rows.append((both + mine)[:max(-(-n // page), 0)])
            lens.append(n)
        if isinstance(e, tuple):
            end = len(lens)
    cu.append(end if cu else 0)
    n_pages = used + 2
    ids = torch.randperm(n_pages, generator=gen, device="cuda").tolist()
    kp, vp = (make_pool(n_pages, g, page, d, dt(kv), tf, gen, math.nan) for _ in range(2))
    for p, k in fills:
        kp[ids[p], :, :k] = (torch.randn(g, k, d, generator=gen, device="cuda") * hot).to(dt(kv))
        vp[ids[p], :, :k] = torch.randn(g, k, d, generator=gen, device="cuda").to(dt(kv))
    width = max([len(r) for r in rows] + [1]) + 1
    table = i32([[ids[p] for p in r] + [2 ** 31 - 1] * (width - len(r)) for r in rows])
    q = (torch.randn(len(lens), h * d, generator=gen, device="cuda") * hot).to(dt(act))
    return kp, vp, table, lens, q, i32(cu), i32(shared)


SHARED_CASES = [
    # groups, heads, kv heads, size, (act, kv), page, tokens_first, hot
    ([(64, [5, 0, 70])], 4, 2, 64, (F32, F32), 16, False, 1.0),
    ([(300, [24, 24, 24, 24])], 16, 16, 128, (F32, F16), 16, False, 1.0),
    ([7, (129, [1, 2]), (40, [3]), (1000, [0, 0, 0]), 0, 90], 28, 4, 64, (F16, F16), 8, True, 1.5),
    ([(2048, [30] * 40)], 32, 4, 128, (BF16, BF16), 64, False, 1.0),
    ([(513, [5] * 9), (100, [700, -40, -99, 3, 0])], 6, 3, 128, (F32, F32), 32, True, 1.0),
    ([(700, [64, 0, 3])], 12, 1, 256, (F16, F16), 32, False, 1.0),
    ([(257, [90, 1])], 16, 1, 256, (F32, F16), 128, True, 1.0),
    ([(640, [129, 1, 2, 90])], 10, 2, 256, (BF16, BF16), 8, False, 1.0),
    ([(400, [33, 2]), (400, [1, 33])], 8, 1, 256, (F32, F32), 16, False, 1.0),
    ([(5, [3, 9]), (0, [4, 4]), (-8, [4, 70])], 8, 2, 64, (F32, F16), 8, False, 1.0),
    ([(3000, [11] * 5)], 100, 1, 128, (F16, F16), 8, True, 2.0),
    ([(256, [128] * 130)], 5, 5, 64, (BF16, BF16), 128, False, 1.0),
    ([(16, [1] * 3)] * 60, 4, 2, 64, (F32, F16), 16, False, 1.0),
    ([(1024, [0, 0])], 8, 8, 128, (F16, F16), 1024, False, 4.0),
    ([(33000, [100, 7])], 8, 2, 128, (F32, F16), 16, False, 1.0),
    ([0, 0, 300, 1], 8, 4, 64, (BF16, BF16), 16, False, 1.0),
    ([(128, [0] * 2), (127, [1] * 2), (136, [8] * 3)], 7, 1, 64, (F32, F16), 8, False, 1.0),
]


@gpu
@pytest.mark.parametrize("case", SHARED_CASES, ids=lambda c: str(c)[:70])
def test_attn_shared(case):
    import torch
    groups, h, g, d, (act, kv), page, tf, hot = case
    negative = any(isinstance(e, tuple) and e[0] < 0 for e in groups)
    plain = [(max(e[0], 0), e[1]) if isinstance(e, tuple) else e for e in groups]
    kp, vp, table, lens, q, cu, shared = make_groups(plain, h, g, d, act, kv, page, tf, 11, hot)
    if negative:
        shared[-1] = -8
    P = V.PagedKV(kp, vp, h, dt(act))
    out = torch.full_like(q, math.nan)
    P.attn_shared(q, table, i32(lens), cu, shared, out)
    if negative:
        with pytest.raises(V.VireoError):
            P.sync()
        shared[-1] = 0  # as it was taken
    P.sync()
    check_attn(out, q, kp, vp, table, lens, h, act, kv, 1 / math.sqrt(d), page)
    again = torch.full_like(q, 1.0)
    P.attn_shared(q.view(len(lens), h, d), table, i32(lens), cu, shared, again.view(len(lens), h, d),
                  scale=1 / math.sqrt(d))
    assert torch.equal(again, out)  # the same bits every time
    # strided rows, another scale, out over q
    wide = torch.zeros(len(lens), h * d + 64, dtype=q.dtype, device="cuda")
    wide[:, :h * d] = q
    P.attn_shared(wide[:, :h * d], table, i32(lens), cu, shared, wide[:, :h * d], scale=-0.05)
    check_attn(wide[:, :h * d], q, kp, vp, table, lens, h, act, kv, -0.05, page)
    assert (wide[:, h * d:] == 0).all()


@gpu
@pytest.mark.parametrize("act,kv", PAIRS)
def test_attn_shared_without_groups_is_attention(act, kv):
    import torch
    kp, vp, table, lens, q, _, _ = make_groups([70, 0, 1, 333], 8, 2, 128, act, kv, 16, False, 4)
    P = V.PagedKV(kp, vp, 8, dt(act))
    out = torch.full_like(q, math.nan)
    P.attn_shared(q, table, i32(lens), i32([2]), i32([]), out)
    P.sync()
    check_attn(out, q, kp, vp, table, lens, 8, act, kv, 1 / math.sqrt(128), 16)
    none = torch.zeros(0, 8 * 128, dtype=q.dtype, device="cuda")
    P.attn_shared(none, table[:0], i32([]), i32([0, 0]), i32([5]), none.clone())
    P.sync()


@gpu
@pytest.mark.parametrize("act,kv", PAIRS)
def test_attn_shared_groups_that_do_not_rise_are_reported(act, kv):
    """cu is taken as the nearest that rises; what is shared is never more than the first request has."""
    import torch
    kp, vp, table, lens, q, cu, shared = make_groups([(64, [5, 9, 80]), (32, [1, 2])], 4, 2, 64, act, kv, 16, False, 4)
    P = V.PagedKV(kp, vp, 4, dt(act))
    for bad in ([0, 3, 9], [-4, 3, 5], [0, 3, 1], [3, 0, 5], [2 ** 31 - 1, -1, 0]):
        out = torch.full_like(q, math.nan)
        P.attn_shared(q, table, i32(lens), i32(bad), shared, out)
        with pytest.raises(V.VireoError) as e:
            P.sync()
        assert e.value.status == -1
        check_attn(out, q, kp, vp, table, lens, 4, act, kv, 0.125, 16)
    out = torch.full_like(q, math.nan)
    P.attn_shared(q, table, i32(lens), cu, i32([2 ** 31 - 1, 47]), out)  # the third request has more than the first
    P.sync()
    want = torch.empty_like(q)
    P.attn_shared(q, table, i32(lens), cu, shared, want)
    check_attn(out[3:], q[3:], kp, vp, table[3:], lens[3:], 4, act, kv, 0.125, 16)


@gpu
@pytest.mark.parametrize("act,kv,d,page", [(F32, F16, 64, 8), (BF16, BF16, 128, 64), (F32, F32, 64, 32),
                                           (F16, F16, 256, 16)])
def test_attn_shared_bad_pages_and_lengths_are_reported(act, kv, d, page):
    """A page number outside the pool reads as zero keys and values, a length beyond the table is cut."""
    import torch
    kp, vp, table, lens, q, cu, shared = make_groups([(4 * page, [page, 2 * page, 3])], 4, 2, d, act, kv, page, False, 3)
    P = V.PagedKV(kp, vp, 4, dt(act))
    table[:, 2] = -1                 # of the prefix
    table[1, 5] = kp.shape[0]        # of one request's own
    table = table[:, :6].contiguous()
    table[2, 5] = table[0, 0]
    kv_len = i32(lens)
    kv_len[2] = 2 ** 31 - 1
    table[2, 4] = table[0, 1]
    out = torch.empty_like(q)
    P.attn_shared(q, table, kv_len, cu, shared, out)
    with pytest.raises(V.VireoError) as e:
        P.sync()
    assert e.value.status == -1
    zk, zv = torch.cat([kp, torch.zeros_like(kp[:1])]), torch.cat([vp, torch.zeros_like(vp[:1])])
    t2 = table.clone()
    t2[(t2 < 0) | (t2 >= kp.shape[0])] = kp.shape[0]
    check_attn(out, q, zk, zv, t2, [lens[0], lens[1], 6 * page], 4, act, kv, 1 / math.sqrt(d), page)
    P.sync()


@gpu
@pytest.mark.parametrize("r", [1, 8])
@pytest.mark.parametrize("act,kv", PAIRS)
def test_attn_shared_infinities(act, kv, r):
    """Keys of -inf scores take no weight, also when they fill whole tiles of
    the prefix; a row of nothing else is zero; a NaN in one request's own
    positions spoils its rows only, one in the prefix its group's only."""
    import torch
    h, g, d, page = 2 * r, 2, 64, 16
    kp, vp, table, lens, q, cu, shared = make_groups([(320, [40, 1, 9]), (160, [3, 0]), 50], h, g, d, act, kv, page,
                                                     False, 5)
    q.copy_(q.abs() + 0.1)
    minus = torch.full((d,), -math.inf, device="cuda").to(kp.dtype)
    for j in range(0, 270):  # of the first group's prefix
        kp[table[0, j // page].item(), :, j % page] = minus
    for j in range(160):     # all of the second's, whose last request has nothing else
        kp[table[3, j // page].item(), :, j % page] = minus
    kp[table[1, 20].item(), 1, 0] = math.nan  # the second request's own position
    P = V.PagedKV(kp, vp, h, dt(act))
    out = torch.full_like(q, 9.0)
    P.attn_shared(q, table, i32(lens), cu, shared, out)
    P.sync()
    for i, skip in ((0, 270), (2, 270), (3, 160), (5, 0)):
        k, v = rows_of(kp, table[i, :-(-lens[i] // page)], lens[i])[:, skip:], rows_of(
            vp, table[i, :-(-lens[i] // page)], lens[i])[:, skip:]
        ref, s = plain_attn(q[i].double().reshape(g, r, d), k, v, 1 / math.sqrt(d))
        err = (out[i].double().reshape(g, r, d) - ref).abs()
        assert (err <= attn_tol(ref, s, float(v.abs().max()), lens[i], d, act, kv)).all(), i
    assert (out[4] == 0).all()
    two = out[1].reshape(g, r, d)
    assert two[0].isfinite().all() and two[1].isnan().all()
    vp[table[0, 19].item(), 0, 5, 7] = math.nan
    P.attn_shared(q, table, i32(lens), cu, shared, out)
    P.sync()
    assert out[:3].reshape(3, g, r, d)[:, 0, :, 7].isnan().all() and out[3:].isfinite().all()


@gpu
@pytest.mark.parametrize("kv", [F32, F16])
def test_attn_shared_sums_do_not_drift(kv):
    """Equal weights over a long prefix: the mean of its values, to fp32's own step a hundred times over."""
    import torch
    n, d, page = 65536, 64, 64
    gen = torch.Generator(device="cuda").manual_seed(2)
    kp = torch.zeros(n // page, 1, page, d, dtype=dt(kv), device="cuda")
    vp = (torch.rand(n // page, 1, page, d, generator=gen, device="cuda") + 0.5).to(dt(kv))
    table = torch.arange(n // page, dtype=torch.int32, device="cuda").expand(3, -1).contiguous()
    q = torch.randn(3, 4 * d, generator=gen, device="cuda")
    P, out = V.PagedKV(kp, vp, 4, torch.float32), torch.empty_like(q)
    P.attn_shared(q, table, i32([n] * 3), i32([0, 3]), i32([n]), out)
    P.sync()
    ref = vp.double().mean((0, 1, 2)).expand(3, 4, d).reshape(3, -1)
    # pieces of at most n positions, added in fp32 to nearest a tile at a time: far below 100 steps
    assert float(((out.double() - ref) / ref).abs().max()) <= 100 * 2.0 ** -24


# ---------------------------------------------------------------------------
# streams, graphs, and all of it together
# ---------------------------------------------------------------------------

@gpu
def test_streams_and_graphs():
    """Each call on a stream of its own, and captured and replayed with other inputs."""
    import torch
    kp, vp, table, lens, q, cu, shared = make_groups([(200, [30, 7, 0])], 8, 2, 64, F32, F16, 16, False, 9)
    P = V.PagedKV(kp, vp, 8, torch.float32)
    kv_len, out, want = i32(lens), torch.zeros_like(q), torch.zeros_like(q)
    logits, score = torch.randn(6, 5000, device="cuda"), torch.zeros(6, device="cuda")
    so, tk, pa, dn = torch.zeros(2, 3, device="cuda"), i32([[0] * 3] * 2), i32([[0] * 3] * 2), i32([[0] * 3] * 2)

    def calls(stream=None):
        P.attn_shared(q, table, kv_len, cu, shared, out, stream=stream)
        V.beam_select(logits, score, 3, score_out=so, token=tk, parent=pa, done_out=dn, stream=stream)
    calls()
    P.sync()
    want.copy_(out)
    first = tk.clone()
    side = torch.cuda.Stream()
    for stream in (side, side.cuda_stream, torch.cuda.default_stream()):
        out.zero_()
        tk.zero_()
        torch.cuda.synchronize()
        calls(stream)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(tk, first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls()
    q.mul_(0.5)
    logits.neg_()
    graph.replay()
    torch.cuda.synchronize()
    check_attn(out, q, kp, vp, table, lens, 8, F32, F16, 0.125, 16)
    best = plain_select(logits, score.cpu(), 3, 3, None, -1)
    assert tk.tolist() == [[f[2] for f in b] for b in best]


@gpu
@pytest.mark.parametrize("act,kv,beams", [(F32, F16, 3), (BF16, BF16, 4)])
def test_a_beam_search(act, kv, beams):
    """Two requests' beam searches over two layers: plan, append, attention over
    what the beams share, the choice, fork and copy, with a compaction on the
    way; against caches that are copied beam by beam."""
    import torch
    torch.manual_seed(3)
    layers, h, g, d, page, n_pages, width, vocab, n = 2, 4, 2, 64, 8, 120, 12, 97, 2
    rows = n * beams
    pools = [[torch.zeros(n_pages, g, page, d, dtype=dt(kv), device="cuda") for _ in range(2)] for _ in range(layers)]
    P = [V.PagedKV(k, v, h, dt(act), rope_dim=0) for k, v in pools]
    new = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
    ring, state = torch.randperm(n_pages, device="cuda").int(), i32([0, n_pages])
    shares, table, other, kv_len = new(n_pages), new(rows, width), new(rows, width), new(rows)
    lens = [[21, 16][i // beams] for i in range(rows)]
    emb, head = torch.randn(vocab, h * d, device="cuda"), torch.randn(h * d, vocab, device="cuda") * 0.3
    wk, wv = torch.randn(layers, h * d, g * d, device="cuda") * 0.06, torch.randn(layers, h * d, g * d, device="cuda") * 0.06
    caches = [[[] for _ in range(rows)] for _ in range(layers)]  # (k, v) of every position

    def step(tokens, seqs):
        """The new tokens' keys and values into pool and caches; q of the last token of each row."""
        total = len(tokens)
        slots, pos, cu, gr = torch.zeros(total, dtype=torch.int64, device="cuda"), new(total), new(rows + 1), new(rows)
        add = i32([seqs.count(i) for i in range(rows)])
        V.kv_plan(kv_len, add, table, ring, state, page, slots=slots, pos=pos, cu=cu, kv_len=kv_len, granted=gr,
                  state_out=state)
        assert gr.all()
        x = emb[torch.tensor(tokens, device="cuda")]
        for l in range(layers):
            k, v, q = (x @ wk[l]).to(dt(act)), (x @ wv[l]).to(dt(act)), x.to(dt(act))
            P[l].append(q, k, v, pos, slots, torch.empty_like(q))
            for t, s in enumerate(seqs):
                caches[l][s].append((k[t].to(dt(kv)), v[t].to(dt(kv))))
        return x

    # the prompts: every beam's row holds its request's prompt once, by a fork of the first row
    first = [i for i in range(rows) if i % beams == 0]
    prompt = [int(t) for i in first for t in torch.randint(0, vocab, (lens[i],))]
    step(prompt, [i for i in first for _ in range(lens[i])])

    def fork(parent):
        nonlocal table, other, caches
        lo, gr, src, dst, rr = new(rows), new(rows), new(rows), new(rows), new(rows)
        V.kv_fork(kv_len, table, parent, shares, ring, state, page, table_out=other, kv_len_out=lo, granted=gr,
                  shares_out=shares, state_out=state, src=src, dst=dst, rows=rr)
        V.kv_copy(P, src, dst, rows=rr)
        assert gr.all()
        kv_len.copy_(lo)
        table, other = other, table
        caches = [[list(c[p]) if p >= 0 else [] for p in parent.tolist()] for c in caches]
    fork(i32([i - i % beams for i in range(rows)]))
    cu, shared = i32([i * beams for i in range(n + 1)]), i32([lens[i * beams] for i in range(n)])
    score = torch.tensor([0.0 if i % beams == 0 else -math.inf for i in range(rows)], device="cuda")
    token = [5] * rows
    for it in range(9):
        x = step(token, list(range(rows)))
        o = x
        for l in range(layers):
            q, out = o.to(dt(act)), torch.empty(rows, h * d, dtype=dt(act), device="cuda")
            P[l].attn_shared(q, table, kv_len, cu, shared, out)
            for i in range(rows):
                k, v = (torch.stack([c[j] for c in caches[l][i]]).view(-1, g, d).transpose(0, 1).double()
                        for j in (0, 1))
                ref, s = plain_attn(q[i].double().view(g, h // g, d), k, v, 1 / math.sqrt(d))
                err = (out[i].double().view(g, h // g, d) - ref).abs()
                assert (err <= attn_tol(ref, s, float(v.abs().max()), k.shape[1], d, act, kv)).all(), (it, l, i)
            o = x + out.float()
        logits = o @ head
        so, tk, pa = torch.zeros(n, beams, device="cuda"), new(n, beams), new(n, beams)
        V.beam_select(logits, score, beams, score_out=so, token=tk, parent=pa)
        want = plain_select(logits, score.cpu(), beams, beams, None, -1)
        assert pa.tolist() == [[f[1] for f in b] for b in want] and tk.tolist() == [[f[2] for f in b] for b in want]
        fork(pa.view(-1))
        score, token = so.view(-1).clone(), tk.flatten().tolist()
        if it == 4:
            src, dst = new(n_pages), new(n_pages)
            V.kv_compact(kv_len, table, ring, page, shares=shares, table_out=table, shares_out=shares, state_out=state,
                         src=src, dst=dst)
            V.kv_copy(P, src, dst)
            held = {p for r, k in zip(table.tolist(), kv_len.tolist()) for p in r[:-(-k // page)]}
            assert max(held) == len(held) - 1 and state.tolist() == [0, n_pages - len(held)]
        # every page is held as often as counted, or free
        held = [p for r, k in zip(table.tolist(), kv_len.tolist()) for p in r[:-(-k // page)]]
        hd, count = state.tolist()
        free = [ring.tolist()[(hd + j) % n_pages] for j in range(count)]
        assert sorted(set(held) | set(free)) == list(range(n_pages)) and len(set(held)) + len(free) == n_pages
        assert all(shares[p].item() == held.count(p) - 1 for p in set(held))
    # the end: everything is given back
    fork(i32([-1] * rows))
    assert state[1].item() == n_pages and not shares.any()
    V.sync()


# ---------------------------------------------------------------------------
# calls that only size, place or company make hard
# ---------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("groups,h,g,d,pair,page", [
    ([(8192, [1] * 64)], 32, 4, 128, (F16, F16), 64),       # stretches that end inside units of 128 rows
    ([(8192, [1] * 64)], 32, 4, 128, (F32, F16), 16),
    ([(256, [0] * 32)] * 30, 32, 4, 128, (BF16, BF16), 64),  # several such units to a stretch
    ([(256, [0, 300] * 16)] * 30, 32, 4, 128, (F32, F16), 64),  # those and small ones in turn
    ([(512, [0] * 40)] * 25, 16, 2, 64, (F32, F16), 32),
    ([(512, [65] * 21)] * 12, 16, 4, 256, (F32, F16), 64),
    ([(3000, [200] * 7), (0, [])] * 2, 16, 2, 256, (BF16, BF16), 8),
    ([(4096, [2] * 40)], 12, 2, 128, (F32, F32), 64),
    ([(256, [3] * 9)] * 30, 8, 2, 256, (F32, F32), 16)])
def test_attn_shared_of_many_rows(groups, h, g, d, pair, page):
    import torch
    act, kv = pair
    kp, vp, table, lens, q, cu, shared = make_groups(groups, h, g, d, act, kv, page, False, 21)
    P, out = V.PagedKV(kp, vp, h, dt(act)), torch.full_like(q, math.nan)
    P.attn_shared(q, table, i32(lens), cu, shared, out)
    P.sync()
    check_attn(out, q, kp, vp, table, lens, h, act, kv, 1 / math.sqrt(d), page)


@gpu
@pytest.mark.parametrize("act,kv", PAIRS)
def test_attn_shared_and_copy_beyond_32_bits_of_a_strided_pool(act, kv):
    """Every other page of a pool of more than 2^32 bytes, its last ones in use."""
    import torch
    kp, vp, table, lens, q, cu, shared = make_groups([(200, [30, 7, 0]), 90], 8, 2, 64, act, kv, 16, False, 9)
    n, m = kp.shape[0], 2 ** 32 // (2 * 2 * 16 * 64 * kp.element_size()) + kp.shape[0]
    big = [torch.empty(2 * m, 2, 16, 64, dtype=dt(kv), device="cuda")[::2] for _ in range(2)]
    assert big[0].stride(0) * (m - n) * kp.element_size() >= 2 ** 32
    for b, x in zip(big, (kp, vp)):
        b[m - n:] = x
        b[:n] = math.nan
    high = torch.where((table >= 0) & (table < n), table + (m - n), table)
    P, out, want = V.PagedKV(*big, 8, dt(act)), torch.full_like(q, math.nan), torch.full_like(q, math.nan)
    P.attn_shared(q, high, i32(lens), cu, shared, out)
    V.PagedKV(kp, vp, 8, dt(act)).attn_shared(q, table, i32(lens), cu, shared, want)
    P.sync()
    assert torch.equal(out, want)
    low = torch.randperm(n, device="cuda").int()  # down and back to other places
    up = torch.arange(m - n, m, device="cuda").int()
    V.kv_copy(P, up, low)
    assert torch.equal(big[0][low.long()].view(torch.uint8), kp.view(torch.uint8))
    for b in big:
        b[m - n:] = 0
    V.kv_copy(P, low, up.flip(0).contiguous())
    P.sync()
    assert torch.equal(big[1][m - n:].flip(0).view(torch.uint8), vp.view(torch.uint8))


@gpu
@pytest.mark.parametrize("t", [F32, F16])
def test_beam_select_beyond_32_bits(t):
    import torch
    vocab, rows, stride = 5000, 6, 900_000_011
    wide = torch.empty(rows * stride, dtype=dt(t), device="cuda").as_strided((rows, vocab), (stride, 1))
    gen = torch.Generator(device="cuda").manual_seed(1)
    wide.copy_(torch.randn(rows, vocab, generator=gen, device="cuda"))
    check_select(wide, torch.zeros(rows, device="cuda"), 3, 5)


@gpu
@pytest.mark.parametrize("rows,beams", [(1, 1), (4, 4), (320, 8)])
@pytest.mark.parametrize("vocab", [30001, 151936])
def test_beam_select_of_rising_and_late_values(rows, beams, vocab):
    """More candidates between two rankings than the list holds, in every chunk and in one."""
    import torch
    if rows > 8 and vocab > 50000:
        rows = 16
    step = torch.arange(vocab, device="cuda", dtype=torch.float32) * 2.0 ** -10
    rising = (step + torch.arange(rows, device="cuda")[:, None] * 2.0 ** -12).contiguous()
    zero = torch.zeros(rows, device="cuda")
    # totals of two rows never meet: steps of 2^-10, rows 0.3 of one apart
    score = (torch.arange(rows, device="cuda") % beams).float() * (-0.3 * 2.0 ** -10)
    check_select(rising, score, beams, min(7, beams * 3))
    late = torch.zeros(rows, vocab, device="cuda")
    late[:, vocab - 9000:vocab - 8000] = 5.0  # of one value: the lower index first
    check_select(late, zero, beams, 32)
    late[:, 20000:20600] = 5.0
    late[0, 20000:20600] = 5.5
    check_select(late, zero, beams, 5)


def share_calls(seed):
    """A call of each kind, with all that it needs: run(stream), and what it wrote."""
    import torch
    kp, vp, table, lens, q, cu, shared = make_groups([(160, [30, 7, 0] * seed), (96, [9] * 4)], 8, 2, 64, F32, F16, 16,
                                                     False, seed)
    P, out, kv_len = V.PagedKV(kp, vp, 8, torch.float32), torch.zeros_like(q), i32(lens)
    logits = torch.randn(6, 9000, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")
    score, so = torch.zeros(6, device="cuda"), torch.zeros(2, 3, device="cuda")
    tk, pa = (torch.zeros(2, 3, dtype=torch.int32, device="cuda") for _ in range(2))
    page, width, n, m = 8, 33, 40 * seed, 50 * seed
    f_len, f_table, parent, keep, shares, ring, state = fork_case(n, m, page, width, seed)
    ft, n_pages = i32(f_table), len(ring)
    new = lambda *s: torch.full(s, 9, dtype=torch.int32, device="cuda")
    a = [i32(f_len), ft, i32(parent), i32(shares), i32(ring), i32(state)]
    b = dict(table_out=new(m, width), kv_len_out=new(m), granted=new(m), shares_out=new(n_pages), state_out=new(2),
             src=new(m), dst=new(m), rows=new(m))
    keeps = i32(keep)
    c = dict(table_out=new(n, width), state_out=new(2), src=new(n_pages), dst=new(n_pages), shares_out=new(n_pages))
    ring2 = new(n_pages)
    pool = [torch.randn(n_pages, 2, page, 64, device="cuda") for _ in range(2)]
    start, C2 = [x.clone() for x in pool], V.PagedKV(*pool, 2, torch.float32)

    def run(stream=None):
        P.attn_shared(q, table, kv_len, cu, shared, out, stream=stream)
        V.beam_select(logits, score, 3, score_out=so, token=tk, parent=pa, stream=stream)
        V.kv_fork(*a, page, keep=keeps, **b, stream=stream)
        V.kv_copy(C2, b["src"], b["dst"], b["rows"], stream=stream)
        V.kv_compact(a[0], ft, ring2, page, shares=a[3], **c, stream=stream)

    def reset():
        for x, y in zip(pool, start):
            x.copy_(y)
    inputs = dict(q=q, logits=logits, keep=keeps)
    return run, reset, inputs, [out, so, tk, pa, ring2] + pool + [a[4]] + list(b.values()) + list(c.values())


@gpu
def test_calls_at_once_on_two_streams():
    import torch
    one, two = share_calls(1), share_calls(3)
    want = []
    for run, reset, _, results in (one, two):
        run()
        torch.cuda.synchronize()
        want.append([x.clone() for x in results])
        reset()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        torch.cuda.synchronize()
        for c, s in zip((one, two), streams):
            c[0](s)
        torch.cuda.synchronize()
        for c, w in zip((one, two), want):
            assert all(torch.equal(x, y) for x, y in zip(c[3], w))
            c[1]()
    V.sync()


@gpu
def test_captured_calls_follow_their_inputs():
    """One graph of every call, replayed with other inputs, against the calls themselves."""
    import torch
    run, reset, inputs, results = share_calls(2)
    ring = results[7]
    ring0 = ring.clone()
    run()
    torch.cuda.synchronize()
    reset()
    ring.copy_(ring0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for _ in range(2):
        inputs["q"].mul_(-0.7)
        inputs["logits"].neg_()
        inputs["keep"].copy_(torch.where(inputs["keep"] > 3, inputs["keep"] - 3, inputs["keep"]))
        run()
        torch.cuda.synchronize()
        want = [x.clone() for x in results]
        reset()
        ring.copy_(ring0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(results, want))
        reset()
        ring.copy_(ring0)
    V.sync()


@gpu
def test_attn_shared_from_two_threads():
    """Calls that need different amounts of shared memory, from threads of their own."""
    import threading

    import torch
    P, work = None, []
    for n, seed in ((3, 1), (5000, 2)):
        kp, vp, table, lens, q, cu, shared = make_groups([(64, [1] * n)], 2, 2, 64, F32, F32, 16, False, seed)
        P = V.PagedKV(kp, vp, 2, torch.float32)
        kv_len, want = i32(lens), torch.zeros_like(q)
        P.attn_shared(q, table, kv_len, cu, shared, want)
        P.sync()
        work.append((P, q, table, kv_len, cu, shared, want))
    failed = []

    def loop(P, q, table, kv_len, cu, shared, want):
        try:
            stream, out = torch.cuda.Stream(), torch.zeros_like(want)
            stream.wait_stream(torch.cuda.default_stream())
            for _ in range(200):
                P.attn_shared(q, table, kv_len, cu, shared, out, stream=stream)
            stream.synchronize()
            if not torch.equal(out, want):
                failed.append("results")
        except Exception as e:  # into the test's own thread
            failed.append(repr(e))
    threads = [threading.Thread(target=loop, args=w) for w in work]
    for x in threads:
        x.start()
    for x in threads:
        x.join()
    assert not failed


@gpu
@pytest.mark.parametrize("seed", range(12))
def test_attn_shared_of_random_groups(seed):
    """Groups and single requests, with and without positions of their own, in any mixture."""
    import torch
    r = random.Random(seed)
    act, kv = PAIRS[seed % len(PAIRS)]
    g, per, d, page = r.choice([1, 2, 4]), r.choice([1, 3, 8, 16, 40]), r.choice([64, 128, 256]), r.choice([8, 16, 64])
    own = lambda: r.choice([0, 0, 1, page, 130, r.randrange(400)])
    groups = [own() for _ in range(r.randrange(4))]  # groups stand in one run
    groups += [(r.choice([0, 5, 16, 100, 512, 2000]), [own() for _ in range(r.randrange(40))])
               for _ in range(r.randrange(1, 25))]
    groups += [own() for _ in range(r.randrange(4))]
    kp, vp, table, lens, q, cu, shared = make_groups(groups, g * per, g, d, act, kv, page, False, seed)
    P, out = V.PagedKV(kp, vp, g * per, dt(act)), torch.full_like(q, math.nan)
    P.attn_shared(q, table, i32(lens), cu, shared, out)
    P.sync()
    check_attn(out, q, kp, vp, table, lens, g * per, act, kv, 1 / math.sqrt(d), page)


@gpu
@pytest.mark.parametrize("n,beams,k,vocab,t", [
    (20, 32, 32, 1000, F32), (3, 16, 32, 7001, F16), (2, 32, 31, 20000, BF16), (1, 1, 32, 150001, F32),
    (5, 17, 17, 600, F32), (1, 9, 16, 4096, F32), (30, 3, 24, 8, F32)])
def test_beam_select_of_many_continuations(n, beams, k, vocab, t):
    """Rows of one distribution, and rows of which one has all of the best."""
    import torch
    gen = torch.Generator(device="cuda").manual_seed(vocab + k)
    logits = (torch.randn(n * beams, vocab, generator=gen, device="cuda") * 3).to(dt(t))
    score = -torch.rand(n * beams, generator=gen, device="cuda")
    check_select(logits, score, beams, k)
    score[::beams] += 60.0
    check_select(logits, score, beams, k)
    score[::beams] -= 55.0
    done = (torch.rand(n * beams, generator=gen, device="cuda") < 0.5).int()
    check_select(logits, score, beams, k, done, vocab - 1)


@gpu
@pytest.mark.parametrize("low", [-3.4028234663852886e38, -1e30])
@pytest.mark.parametrize("beams,vocab,k", [(4, 4, 16), (16, 2, 32), (4, 9, 32), (3, 20, 24), (32, 1, 32), (4, 5000, 32)])
def test_beam_select_of_large_finite_scores(beams, vocab, k, low):
    """Beams not begun yet have a large finite score in place of -inf: their totals
    are one value whatever their tokens, and none may get lost."""
    import torch
    n = 24
    gen = torch.Generator(device="cuda").manual_seed(vocab)
    logits = torch.randn(n * beams, vocab, generator=gen, device="cuda") * 2
    for begun in (1, 0):  # the first beam of each request, or none
        score = torch.full((n, beams), low, device="cuda")
        score[:, :begun] = 0.0
        so = torch.full((n, k), 7.0, device="cuda")
        token, parent = i32([[99] * k] * n), i32([[99] * k] * n)
        V.beam_select(logits, score.flatten(), beams, score_out=so, token=token, parent=parent)
        V.sync()
        for i in range(n):
            got = list(zip(parent[i].tolist(), token[i].tolist()))
            assert len(set(got)) == k, i
            assert all(i * beams <= p < (i + 1) * beams and 0 <= t < vocab for p, t in got), i
            first = min(k, vocab) if begun else 0
            best = torch.argsort(logits[i * beams], descending=True, stable=True)[:first].tolist()
            assert got[:first] == [(i * beams, t) for t in best], i
            assert so[i, first:].tolist() == [pytest.approx(low, rel=2.0 ** -24)] * (k - first), i


@gpu
@pytest.mark.parametrize("far", [1e5, 3e6, 1e8, 3e9, 7e9, 1e12, 9e29, 2e30])
@pytest.mark.parametrize("t", [F32, BF16])
def test_beam_select_of_logits_far_from_zero(far, t):
    """Rows that a large value has been added to or taken from, as a mask of finite
    values does to all of a row: the logits' differences are what counts."""
    import torch
    n, vocab, k = 6, 5000, 7
    gen = torch.Generator(device="cuda").manual_seed(3)
    for sign in (1.0, -1.0):
        base = torch.tensor([sign * far * (1 + i / 16) for i in range(n)], device="cuda").to(dt(t)).float()
        step = torch.finfo(dt(t)).eps * far * 4  # of the type, there and a little further
        logits = (base[:, None] + step * torch.randint(-20, 1, (n, vocab), generator=gen, device="cuda")).to(dt(t))
        so = torch.full((n, k), 7.0, device="cuda")
        token, parent, dn = (i32([[99] * k] * n) for _ in range(3))
        V.beam_select(logits, torch.zeros(n, device="cuda"), 1, score_out=so, token=token, parent=parent, done_out=dn)
        V.sync()
        x = logits.double()
        top = x.amax(1, keepdim=True)
        less = torch.log(torch.exp(x - top).sum(1, keepdim=True))
        best, ids = torch.sort(x, dim=1, descending=True, stable=True)
        assert torch.equal(token.long(), ids[:, :k])
        assert parent.tolist() == [[i] * k for i in range(n)] and (dn == 0).all()
        want = best[:, :k] - top - less
        # and in 64 bits log sum exp, its sum with the largest and the total's two are rounded at the logits' size
        tol = 2.0 ** -24 * want.abs() + 2.0 ** -19 + 4 * 2.0 ** -53 * x.abs().amax(1, keepdim=True)
        assert ((so.double() - want).abs() <= tol).all(), float(((so.double() - want).abs() / tol).max())


@gpu
@pytest.mark.parametrize("r", [1, 8, 40])
@pytest.mark.parametrize("act,kv", PAIRS)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_attn_shared_of_large_scores(act, kv, d, r):
    """Scores of which each differs from the next by more than any weight can tell:
    the position with the largest takes it all, in the prefix or behind it,
    however large the scores are."""
    import torch
    h, g, page = 2 * r, 2, 16
    kp, vp, table, lens, q, cu, shared = make_groups([(160, [40, 0, 7])], h, g, d, act, kv, page, False, 6)
    order = torch.randperm(256, generator=torch.Generator().manual_seed(1)).tolist()
    unit = 128.0 if act == F16 else 2.0 ** -8  # keys 1 .. 256 times that, every type's own
    best = []
    for i, n in enumerate(lens):
        for j in range(n):
            p = table[i, j // page].item()
            kp[p, :, j % page] = 0
            kp[p, :, j % page, 3] = order[j if j < 160 else j + 40 * (i == 2)] * unit
        k, v = rows_of(kp, table[i, :-(-n // page)], n), rows_of(vp, table[i, :-(-n // page)], n)
        best.append(v[:, k[0, :, 3].argmax()])
    want = torch.stack(best)[:, :, None].expand(-1, -1, r, -1)
    # errors of scores (the bound's third argument) change nothing: other weights stay zero
    tol = attn_tol(want, 0.0, float(want.abs().max()), max(lens), d, act, kv)
    P, out = V.PagedKV(kp, vp, h, dt(act)), torch.empty_like(q)
    some = 1.0 + torch.rand(len(lens), h, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda") * 0.9
    for e in (10, 12, 14) if act == F16 else (17, 20, 22, 24, 26, 30, 40, 80, 116, 125):
        for scale in (0.125, -0.125):
            q.zero_()
            q.view(len(lens), h, d)[:, :, 3] = some * math.copysign(2.0 ** e, scale)
            P.attn_shared(q, table, i32(lens), cu, shared, out, scale=scale)
            P.sync()
            err = (out.view(len(lens), g, r, d).double() - want).abs()
            assert (err <= tol).all(), (e, scale, float((err / tol).max()))


@gpu
@pytest.mark.parametrize("t", [F32, BF16])
def test_beam_select_scores_in_any_company(t):
    """A row's scores alone, among others, at another alignment and beside a row like
    it: each time within 2^-19 of 64 bits and the rounding, and the same in every call."""
    import torch
    vocab, k = 20011, 5
    gen = torch.Generator(device="cuda").manual_seed(9)
    row = (torch.randn(vocab, generator=gen, device="cuda") * 3).to(dt(t))
    other = (torch.randn(vocab, generator=gen, device="cuda") * 3).to(dt(t))
    want = torch.sort(row.double() - torch.logsumexp(row.double(), 0), descending=True).values[:k]
    shifted = torch.zeros(3, vocab + 3, device="cuda").to(dt(t))[:, 3:]
    shifted.copy_(row.expand(3, -1))
    for logits, beams, far in ((row[None], 1, 0.0), (torch.stack([row] + [other] * 7), 8, 40.0), (shifted, 1, 0.0),
                               (torch.stack([row] * 2), 2, 0.0), (row.expand(700, -1).contiguous(), 1, 0.0)):
        n = logits.shape[0] // beams
        score = torch.zeros(n, beams, device="cuda")
        score[:, 1:] -= far
        got = []
        for _ in range(2):
            so, token, parent = torch.zeros(n, k, device="cuda"), i32([[0] * k] * n), i32([[0] * k] * n)
            V.beam_select(logits, score.flatten(), beams, score_out=so, token=token, parent=parent)
            V.sync()
            got.append(so)
        assert torch.equal(got[0], got[1])
        best = want if beams != 2 else want.repeat_interleave(2)[:k]
        assert ((so.double() - best).abs() <= 2.0 ** -24 * best.abs() + 2.0 ** -19).all()


@gpu
@pytest.mark.parametrize("act,kv", PAIRS)
def test_attn_shared_of_more_than_the_first_request_has(act, kv):
    """shared beyond the first request's length, or not in whole pages, is the whole pages that
    the first request has: every row, the group's own among them, comes out as with those."""
    import torch
    kp, vp, table, lens, q, cu, shared = make_groups([(64, [5, 9, 80]), (32, [1, 2])], 4, 2, 64, act, kv, 16, False, 4)
    P = V.PagedKV(kp, vp, 4, dt(act))
    want = torch.full_like(q, math.nan)
    P.attn_shared(q, table, i32(lens), cu, shared, want)
    check_attn(want, q, kp, vp, table, lens, 4, act, kv, 0.125, 16)
    for more in ([2 ** 31 - 1, 47], [79, 2 ** 31 - 1], [70, 33], [64, 32]):
        out = torch.full_like(q, math.nan)
        P.attn_shared(q, table, i32(lens), cu, i32(more), out)
        P.sync()
        assert torch.equal(out, want), more


@gpu
@pytest.mark.parametrize("r", [1, 12])
@pytest.mark.parametrize("act,kv", [(F32, F32), (F32, F16), (BF16, BF16)])
def test_attn_shared_of_scales_below_the_normal_numbers(act, kv, r):
    """A scale of 2^-128 against queries of 2^127: scores of up to 1, as with 1 and 1; keys of
    -inf, whose scores that scale must not turn into anything else, take no weight."""
    import torch
    h, g, d, page = r, 1, 64, 16
    kp, vp, table, lens, q, cu, shared = make_groups([(160, [40, 0, 7])], h, g, d, act, kv, page, False, 8)
    for i, n in enumerate(lens):
        for j in range(n):
            p = table[i, j // page].item()
            kp[p, :, j % page] = 0
            kp[p, :, j % page, 3] = (j * 97 % 256) / 256
    P, out = V.PagedKV(kp, vp, h, dt(act)), torch.empty_like(q)
    q.zero_()
    q.view(len(lens), h, d)[:, :, 3] = 1.875 * 2.0 ** 127
    P.attn_shared(q, table, i32(lens), cu, shared, out, scale=2.0 ** -128)
    P.sync()
    check_attn(out, q, kp, vp, table, lens, h, act, kv, 2.0 ** -128, page)
    for j in range(5, 160):
        kp[table[0, j // page].item(), :, j % page, 3] = -math.inf
    P.attn_shared(q, table, i32(lens), cu, shared, out, scale=2.0 ** -128)
    P.sync()
    for i, n in enumerate(lens):
        live = [j for j in range(n) if j < 5 or j >= 160]
        k, v = (rows_of(x, table[i, :-(-n // page)], n)[:, live] for x in (kp, vp))
        ref, s = plain_attn(q[i].double().reshape(g, r, d), k, v, 2.0 ** -128)
        err = (out[i].double().reshape(g, r, d) - ref).abs()
        assert (err <= attn_tol(ref, s, float(v.abs().max()), n, d, act, kv)).all(), i


@gpu
@pytest.mark.parametrize("n,m,width", [(64, 70, 40), (700, 900, 30)])
def test_fork_that_refused_rows_can_be_given_up(n, m, width):
    """With shares_out and state_out apart the next call, from the old state, is as if there
    had been none; with as many free pages as rows none is refused."""
    page = 8
    kv_len, table, parent, keep, shares, ring, state = fork_case(n, m, page, width, 5, True)
    free = lambda ring, state: [ring[(state[0] + j) % len(ring)] for j in range(state[1])]
    got = run_fork(kv_len, table, parent, keep, shares, ring, state, page, width)
    granted, after = got[2], got[4]
    assert 0 in granted and free(after, state) == free(ring, state)
    # the refused ones end instead
    fewer = [p if ok else -1 for p, ok in zip(parent, granted)]
    got = run_fork(kv_len, table, fewer, keep, shares, after, state, page, width)
    want = plain_fork(kv_len, table, fewer, keep, shares, list(ring), state, page, [[-9] * width for _ in fewer])
    for name, a, b in zip(FORK_NAMES, got, want):
        assert (free(a, got[5]) == free(b, want[5])) if name == "ring" else a == b, name
    # m free pages
    n_pages = len(ring) + m
    wide = [-3] * n_pages
    for j in range(m):
        wide[(n_pages - 3 + j) % n_pages] = len(ring) + j
    got = run_fork(kv_len, table, parent, keep, shares + [0] * m, wide, [n_pages - 3, m], page, width)
    assert all(got[2])
    V.sync()


@gpu
def test_beam_select_totals_beyond_fp32():
    """A total that 64 bits hold and fp32 does not is a continuation of score -inf, behind all others."""
    import torch
    low = torch.finfo(torch.float32).min
    x = torch.zeros(2, 40, device="cuda")
    x[:, 1::2] = low
    so, token, parent = torch.zeros(1, 32, device="cuda"), i32([[0] * 32]), i32([[0] * 32])
    V.beam_select(x, torch.tensor([low, -math.inf], device="cuda"), 2, score_out=so, token=token, parent=parent)
    V.sync()
    assert token[0].tolist() == list(range(0, 40, 2)) + list(range(1, 25, 2)) and (parent == 0).all()
    assert (so[0, :20] == low).all() and (so[0, 20:] == -math.inf).all()
