"""The paged key-value operators, as they are measured: cases, inputs, one pass.

Four operators serve many requests from one pool of key-value pages:

* ``plan``: block tables and slot maps from request lengths;
* ``append``: bias, per-head or full-width QK norm and rotation of the new
  tokens' queries and keys, with keys and values written to their slots
  (and the mean key of every page that this fills);
* ``attn``: one new token per request over its pages;
* ``topk``: the same over the first pages, the last pages and the pages
  whose mean key scores highest against the request's queries.

``run`` computes them with elementary torch operations, or (``own``) with
the calls that a program makes of vireo_b200.
"""
import math
import random

import torch

own = False

F32, F16, BF16 = "f32", "f16", "bf16"
DTYPE = {F32: torch.float32, F16: torch.float16, BF16: torch.bfloat16}
# activation and cache types that go together
PAIRS = [(F32, F32), (F32, F16), (F16, F16), (BF16, BF16)]
EPS, ROPE_BASE = 1e-6, 1000000.0


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # a decode step of 64 requests: every one gets one token, one in sixteen needs a page
        dict(name="plan_decode", op="plan", n_seq=64, page=16, ctx=8192, new=1, prompts=0.0, ends=0.0, pad=0),
        # a step that admits prompts, ends requests and is padded to a captured size
        dict(name="plan_mixed", op="plan", n_seq=512, page=16, ctx=4096, new=1024, prompts=0.25, ends=0.1, pad=1000),
        # one token of the 16-head model: full-width norms, f32 activations over an f16 cache
        dict(name="append_one", op="append", n_tok=1, heads=16, kv_heads=16, size=128, act=F32, kv=F16, page=16,
             norm="full", bias=False, rope=128, means=False, tokens_first=False),
        # a prompt batch of the 32 / 4-head model: per-head norms, page means kept for block selection
        dict(name="append_prompt", op="append", n_tok=8192, heads=32, kv_heads=4, size=128, act=BF16, kv=BF16,
             page=64, norm="head", bias=False, rope=128, means=True, tokens_first=False),
        # an odd token count, biases in place of norms, half the dimensions turned, a pool with positions before heads
        dict(name="append_odd", op="append", n_tok=777, heads=14, kv_heads=2, size=64, act=F16, kv=F16, page=16,
             norm="none", bias=True, rope=32, means=False, tokens_first=True),
        # latency: one short request
        dict(name="attn_short", op="attn", n_seq=1, ctx=300, heads=16, kv_heads=16, size=128, act=F32, kv=F16,
             page=16, tokens_first=False),
        # one request of the 32 / 4-head model after an 8192-token prompt
        dict(name="attn_one_long", op="attn", n_seq=1, ctx=8200, heads=32, kv_heads=4, size=128, act=F32, kv=F16,
             page=64, tokens_first=False),
        # a ragged batch, one row of it empty
        dict(name="attn_batch", op="attn", n_seq=64, ctx=8192, heads=32, kv_heads=4, size=128, act=BF16, kv=BF16,
             page=16, tokens_first=False),
        # the cache at the reference's width
        dict(name="attn_f32", op="attn", n_seq=4, ctx=4097, heads=16, kv_heads=16, size=128, act=F32, kv=F32,
             page=32, tokens_first=False),
        # many short requests, seven heads to a key head, small pages, positions before heads
        dict(name="attn_many_short", op="attn", n_seq=128, ctx=1001, heads=28, kv_heads=4, size=64, act=F16, kv=F16,
             page=8, tokens_first=True),
        # block selection in one very long request
        dict(name="topk_one_long", op="topk", n_seq=1, ctx=131085, heads=32, kv_heads=4, size=128, act=BF16, kv=BF16,
             page=64, sink=1, window=4, top=64, tokens_first=False),
        # a ragged batch of long requests with small pages
        dict(name="topk_batch", op="topk", n_seq=16, ctx=32768, heads=32, kv_heads=4, size=128, act=F32, kv=F16,
             page=32, sink=2, window=8, top=48, tokens_first=True),
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_once(rng):
    op = rng.choice(["plan", "append", "attn", "attn", "topk", "topk"])
    if op == "plan":
        return dict(op=op, n_seq=_log(rng, 1, 1024), page=rng.choice([8, 16, 32, 64]), ctx=_log(rng, 64, 8192),
                    new=_log(rng, 1, 1024), prompts=rng.uniform(0.0, 0.5), ends=rng.uniform(0.0, 0.3),
                    pad=rng.randrange(0, 200))
    size = rng.choice([64, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8, 16])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 8, 12, 16])
    act, kv = rng.choice(PAIRS)
    case = dict(op=op, heads=heads, kv_heads=kv_heads, size=size, act=act, kv=kv,
                tokens_first=rng.random() < 0.5)
    if op == "append":
        case.update(n_tok=_log(rng, 1, 8192), page=rng.choice([8, 16, 32, 64, 128]),
                    norm=rng.choice(["none", "head", "full"]), bias=rng.random() < 0.3,
                    rope=rng.choice([0, 32, size // 2, size, size]), means=rng.random() < 0.5)
    elif op == "attn":
        case.update(n_seq=_log(rng, 1, 128), ctx=_log(rng, 1, 16384), page=rng.choice([8, 16, 32, 64, 128]))
    else:
        case.update(n_seq=_log(rng, 1, 16), ctx=_log(rng, 64, 131072), page=rng.choice([16, 32, 64]),
                    sink=rng.randrange(0, 5), window=rng.randrange(1, 9), top=_log(rng, 1, 128))
    return case


def draw(rng):
    most = max(work(c)["bytes"] for c in listed())
    while True:
        case = _draw_once(rng)
        w = work(case)
        # the cost of the plain form goes by the values it handles, however few bytes hold them
        if w["bytes"] <= most and _values(case) <= 300_000_000:
            return case


def _values(case):
    """Values of one of the two pools, every request taken as the longest."""
    if case["op"] in ("plan", "append"):
        return 0
    return case["n_seq"] * case["ctx"] * case["kv_heads"] * case["size"]


def _lengths(n, most, empty):
    """n lengths up to `most`, evenly spread, the longest among them and (from
    four on, if asked) an empty one."""
    golden = 0.6180339887498949
    out = [max(1, int(round(most * ((i * golden) % 1.0)))) if i else most for i in range(n)]
    if empty and n >= 4:
        out[2] = 0
    return out


def _pages(length, page):
    return -(-length // page)


def _plan_requests(case):
    """(past, add) of every request, before they are shuffled."""
    n = case["n_seq"]
    past = _lengths(n, case["ctx"], True)
    fresh, ends = int(n * case["prompts"]), int(n * case["ends"])
    new = _lengths(max(fresh, 1), case["new"], False)
    add = [1] * n
    for i in range(fresh):
        past[n - 1 - i], add[n - 1 - i] = 0, new[i]
    for i in range(ends):
        add[i] = -1
    return past, add


def _table_width(case):
    if case["op"] == "plan":
        return _pages(case["ctx"] + case["new"] + 1, case["page"])
    return _pages(case["ctx"], case["page"])


def _pool_pages(case):
    """Pages of the pool: those in use and a few more."""
    if case["op"] == "plan":
        past, add = _plan_requests(case)
        return sum(_pages(p + max(a, 0), case["page"]) for p, a in zip(past, add)) + 64
    if case["op"] == "append":
        return 2 * _pages(case["n_tok"], case["page"]) + 8
    return sum(_pages(x, case["page"]) for x in _lengths(case["n_seq"], case["ctx"], True)) + 16


def _chosen(case, length):
    """(pages, positions) that block selection attends to."""
    n = _pages(length, case["page"])
    sel = min(n, case["sink"] + case["window"] + case["top"])
    return sel, length - (n - sel) * case["page"]


def work(case):
    if case["op"] == "plan":
        past, add = _plan_requests(case)
        page, n = case["page"], len(past)
        tokens = sum(a for a in add if a > 0)
        fresh = sum(_pages(p + a, page) - _pages(p, page) for p, a in zip(past, add) if a > 0)
        ended = sum(_pages(p, page) for p, a in zip(past, add) if a < 0)
        tails = sum(1 for p, a in zip(past, add) if a > 0 and p % page)
        ints = 2 * n + fresh + ended + tails + 2  # read
        ints += fresh + ended + 3 * n + 3 + 3 * (tokens + case["pad"])  # written; a slot is 8 bytes
        return {"bytes": 4 * ints, "flops": 4 * (tokens + n)}
    h, g, d = case["heads"], case["kv_heads"], case["size"]
    a, c = DTYPE[case["act"]].itemsize, DTYPE[case["kv"]].itemsize
    if case["op"] == "append":
        t = case["n_tok"]
        moved = t * (2 * h * d * a + 2 * g * d * (a + c) + 12)
        if case["means"]:
            moved += (t // case["page"]) * g * d * c
        flops = t * d * ((h + g) * (3 * (case["rope"] > 0) + 4 * (case["norm"] != "none"))
                         + (h + 2 * g) * case["bias"] + g * case["means"])
        return {"bytes": moved, "flops": flops}
    lens = _lengths(case["n_seq"], case["ctx"], True)
    moved, flops = 0, 0
    for x in lens:
        moved += 2 * h * d * a + 4
        if case["op"] == "topk":
            n = _pages(x, case["page"])
            sel, x = _chosen(case, x)
            scored = max(0, n - case["sink"] - case["window"]) if n > sel else 0
            moved += scored * g * d * c + g * (case["sink"] + case["window"] + case["top"]) * 4
            flops += 2 * scored * h * d
            moved += n * 4
        else:
            moved += _pages(x, case["page"]) * 4
        moved += x * 2 * g * d * c
        flops += 4 * x * h * d
    return {"bytes": moved, "flops": flops}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype).cuda()


def _pool(case, n_pages, gen):
    """A pool seen as [page, head, position, dim], whichever of heads and positions lies outside."""
    g, p, d = case["kv_heads"], case["page"], case["size"]
    dtype = DTYPE[case["kv"]]
    if case["tokens_first"]:
        return torch.randn(n_pages, p, g, d, generator=gen, device="cuda", dtype=dtype).transpose(1, 2)
    return torch.randn(n_pages, g, p, d, generator=gen, device="cuda", dtype=dtype)


def prepare(case, seed):
    rng = random.Random(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    if case["op"] == "plan":
        _prepare_plan(case, rng, state)
    elif case["op"] == "append":
        _prepare_append(case, rng, gen, state)
    else:
        _prepare_attn(case, rng, gen, state)
    if own and case["op"] != "plan":
        import vireo_b200
        state["kv"] = vireo_b200.PagedKV(state["kpool"], state["vpool"], case["heads"], DTYPE[case["act"]], eps=EPS,
                                         rope_base=ROPE_BASE, rope_dim=case.get("rope", case["size"]))
    return state


def _prepare_plan(case, rng, state):
    past, add = _plan_requests(case)
    order = list(range(len(past)))
    rng.shuffle(order)
    past, add = [past[i] for i in order], [add[i] for i in order]
    n_pages, width, page = _pool_pages(case), _table_width(case), case["page"]
    ids = list(range(n_pages))
    rng.shuffle(ids)
    rows = [[-1] * width for _ in past]
    used = 0
    for row, p in zip(rows, past):
        k = _pages(p, page)
        row[:k] = ids[used:used + k]
        used += k
    free = ids[used:]
    head = rng.randrange(n_pages)
    ring = [-1] * n_pages
    for i, p in enumerate(free):
        ring[(head + i) % n_pages] = p
    tokens = sum(a for a in add if a > 0) + case["pad"]
    new = lambda n, dtype=torch.int32: torch.zeros(n, dtype=dtype, device="cuda")
    state.update(past=_ints(past), add=_ints(add), table=_ints(rows), ring=_ints(ring),
                 free=_ints([head, len(free)]), slots=new(tokens, torch.int64), pos=new(tokens), cu=new(len(past) + 1),
                 kv_len=new(len(past)), granted=new(len(past)), free_out=new(2))


def _prepare_append(case, rng, gen, state):
    t, h, g, d = case["n_tok"], case["heads"], case["kv_heads"], case["size"]
    n_pages = _pool_pages(case)
    # q | k | v as one projection leaves them: rows of one buffer
    qkv = torch.randn(t, (h + 2 * g) * d, generator=gen, device="cuda").to(DTYPE[case["act"]])
    vec = lambda n, mean, std: torch.randn(n, generator=gen, device="cuda") * std + mean
    full = case["norm"] == "full"
    # requests of several lengths, each at its own position and in its own pages
    pos, slots = [], []
    ids = list(range(n_pages))
    rng.shuffle(ids)
    used = 0
    while len(pos) < t and used < n_pages:
        n = min(t - len(pos), rng.randrange(1, max(2, t // 2 + 1)))
        n = min(n, (n_pages - used) * case["page"])
        first = rng.randrange(0, 30000) // case["page"] * case["page"]
        for j in range(n):
            pos.append(first + j)
            slots.append(ids[used + j // case["page"]] * case["page"] + j % case["page"])
        used += _pages(n, case["page"])
        if n_pages - used <= _pages(t - len(pos), case["page"]):
            break
    while len(pos) < t:  # the rest as one request
        j = 0
        first = rng.randrange(0, 30000) // case["page"] * case["page"]
        while len(pos) < t:
            pos.append(first + j)
            slots.append(ids[used + j // case["page"]] * case["page"] + j % case["page"])
            j += 1
    state.update(q=qkv[:, :h * d], k=qkv[:, h * d:(h + g) * d], v=qkv[:, (h + g) * d:], pos=_ints(pos),
                 slots=_ints(slots, torch.int64), kpool=_pool(case, n_pages, gen), vpool=_pool(case, n_pages, gen),
                 q_out=torch.zeros(t, h * d, device="cuda", dtype=DTYPE[case["act"]]))
    state["q_norm"] = vec(h * d if full else d, 1.0, 0.1) if case["norm"] != "none" else None
    state["k_norm"] = vec(g * d if full else d, 1.0, 0.1) if case["norm"] != "none" else None
    for name, n in (("bq", h * d), ("bk", g * d), ("bv", g * d)):
        state[name] = vec(n, 0.0, 0.3) if case["bias"] else None
    state["means"] = torch.zeros(n_pages, g, d, device="cuda", dtype=DTYPE[case["kv"]]) if case["means"] else None
    page = case["page"]
    # which pages this fills: those that get a token at their last position
    state["filled"] = _ints(sorted({s // page for s in slots if s % page == page - 1}), torch.int64)


def _prepare_attn(case, rng, gen, state):
    n_seq, h, d, page = case["n_seq"], case["heads"], case["size"], case["page"]
    lens = _lengths(n_seq, case["ctx"], True)
    rng.shuffle(lens)
    n_pages, width = _pool_pages(case), _table_width(case)
    kpool, vpool = _pool(case, n_pages, gen), _pool(case, n_pages, gen)
    # keys of one page resemble one another, as neighbouring tokens' do
    kpool.mul_(0.8).add_(torch.randn(n_pages, case["kv_heads"], 1, d, generator=gen, device="cuda",
                                     dtype=kpool.dtype) * 0.6)
    ids = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((n_seq, width), -1, dtype=torch.int32, device="cuda")
    used = 0
    for i, x in enumerate(lens):
        k = _pages(x, page)
        table[i, :k] = ids[used:used + k]
        used += k
    act = DTYPE[case["act"]]
    state.update(lens=lens, kv_len=_ints(lens), table=table, kpool=kpool, vpool=vpool,
                 q=torch.randn(n_seq, h * d, generator=gen, device="cuda").to(act),
                 out=torch.zeros(n_seq, h * d, device="cuda", dtype=act))
    if case["op"] == "topk":
        state["means"] = kpool.float().mean(2).to(kpool.dtype).contiguous()
        n = case["sink"] + case["window"] + case["top"]
        state["sel"] = torch.zeros(n_seq, case["kv_heads"], n, dtype=torch.int32, device="cuda")


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return _own(op, state)
    return {"plan": _plain_plan, "append": _plain_append, "attn": _plain_attn, "topk": _plain_topk}[op](state)


def _plan_outputs(s):
    return [s[n] for n in ("table", "ring", "slots", "pos", "cu", "kv_len", "granted", "free_out")]


def _append_outputs(s):
    return [s["q_out"], s["kpool"], s["vpool"]] + ([s["means"]] if s["means"] is not None else [])


def _own(op, s):
    c = s["case"]
    if op == "plan":
        import vireo_b200
        vireo_b200.kv_plan(s["past"], s["add"], s["table"], s["ring"], s["free"], c["page"], slots=s["slots"],
                           pos=s["pos"], cu=s["cu"], kv_len=s["kv_len"], granted=s["granted"], state_out=s["free_out"])
        return _plan_outputs(s)
    if op == "append":
        s["kv"].append(s["q"], s["k"], s["v"], s["pos"], s["slots"], s["q_out"], q_norm=s["q_norm"],
                       k_norm=s["k_norm"], bq=s["bq"], bk=s["bk"], bv=s["bv"], means=s["means"])
        return _append_outputs(s)
    if op == "attn":
        s["kv"].attn(s["q"], s["table"], s["kv_len"], s["out"])
        return s["out"]
    s["kv"].attn_topk(s["q"], s["table"], s["kv_len"], s["means"], c["sink"], c["window"], c["top"], s["out"],
                      sel=s["sel"])
    return [s["out"], s["sel"]]


def _plain_plan(s):
    page, past, add = s["case"]["page"], s["past"].long(), s["add"].long()
    table, ring, cap = s["table"], s["ring"], s["slots"].shape[0]
    n_pages, width = ring.shape[0], table.shape[1]
    head, count = s["free"][0].long(), s["free"][1].long()
    have = (past + page - 1) // page
    want = (past + add.clamp(min=0) + page - 1) // page
    ok = (past >= 0) & (add >= -1) & (want <= width)
    need = torch.where(ok, want - have, 0)
    ask = torch.where(ok, add.clamp(min=0), 0)
    upto = need.cumsum(0)
    granted = ok & ((need == 0) | (upto <= count)) & ((ask == 0) | (ask.cumsum(0) <= cap))
    got = torch.where(granted, ask, 0)
    cu = torch.cat([got.new_zeros(1), got.cumsum(0)])
    # new pages: table column j of request i, taken from the ring in order
    col = torch.arange(width, device=past.device)
    fresh = granted[:, None] & (add[:, None] > 0) & (col >= have[:, None]) & (col < want[:, None])
    rank = (upto - need)[:, None] + col - have[:, None]
    table.copy_(torch.where(fresh, ring[(head + rank) % n_pages], table))
    taken = torch.where(granted, need, 0).sum()
    # ended requests give their pages back behind the last free one; the
    # entries that get none go to a place past the ring
    ended = granted[:, None] & (add[:, None] == -1) & (col < have[:, None])
    back = ended.flatten().long().cumsum(0)
    at = torch.where(ended.flatten(), (head + count + back - 1) % n_pages, n_pages)
    ring.copy_(torch.cat([ring, ring[:1]]).scatter(0, at, table.flatten())[:n_pages])
    # tokens
    t = torch.arange(cap, device=past.device)
    seq = torch.searchsorted(cu, t, right=True) - 1
    live = t < cu[-1]
    seq = torch.where(live, seq, 0)
    pos = torch.where(live, past[seq] + t - cu[seq], 0)
    slots = table[seq, torch.where(live, pos // page, 0)].long() * page + pos % page
    s["slots"].copy_(torch.where(live, slots, -1))
    s["pos"].copy_(pos)
    s["cu"].copy_(cu)
    s["kv_len"].copy_(torch.where(granted & (add == -1), 0, past + got).clamp(min=0))
    s["granted"].copy_(granted)
    s["free_out"].copy_(torch.stack([(head + taken) % n_pages, count - taken + back[-1]]))
    return _plan_outputs(s)


def _turn(x, pos, rope):
    """Rotates the first `rope` dimensions of x [t, heads, size]: pairs (j, j + rope / 2)."""
    if not rope:
        return x
    half = rope // 2
    freq = ROPE_BASE ** (-torch.arange(half, device=x.device, dtype=torch.float64) * 2 / rope)
    angle = pos.double()[:, None, None] * freq
    c, n = angle.cos().float(), angle.sin().float()
    a, b = x[..., :half], x[..., half:rope]
    return torch.cat([a * c - b * n, a * n + b * c, x[..., rope:]], -1)


def _plain_append(s):
    c = s["case"]
    t, h, g, d, page = c["n_tok"], c["heads"], c["kv_heads"], c["size"], c["page"]

    def head(x, bias, norm, heads):
        x = x.float()
        if bias is not None:
            x = x + bias
        x = x.reshape(t, heads, d)
        if norm is not None:
            w = norm.reshape(-1, d)
            dims = (-1,) if w.shape[0] == 1 and c["norm"] == "head" else (-2, -1)
            x = x / torch.sqrt((x * x).mean(dims, keepdim=True) + EPS) * w
        return x

    q = _turn(head(s["q"], s["bq"], s["q_norm"], h), s["pos"], c["rope"])
    k = _turn(head(s["k"], s["bk"], s["k_norm"], g), s["pos"], c["rope"])
    v = head(s["v"], s["bv"], None, g)
    at, off = s["slots"] // page, s["slots"] % page
    s["q_out"].copy_(q.reshape(t, h * d))
    s["kpool"][at, :, off] = k.to(s["kpool"].dtype)
    s["vpool"][at, :, off] = v.to(s["vpool"].dtype)
    if s["means"] is not None:
        s["means"][s["filled"]] = s["kpool"][s["filled"]].float().mean(2).to(s["kpool"].dtype)
    return _append_outputs(s)


def _attend(q, k, v, live):
    """q [s, g, r, d], k and v [s, g, n, d]; live [s, g or 1, n]: which positions count."""
    q, k, v, live = q.float(), k.float(), v.float(), live[:, :, None]
    w = q @ k.transpose(2, 3) * (1.0 / math.sqrt(q.shape[-1]))
    w = torch.where(live, w, -math.inf)
    w = torch.where(live, torch.exp(w - w.amax(-1, keepdim=True)), 0.0)
    total = w.sum(-1, keepdim=True)
    return torch.where(total > 0, w @ v / total, 0.0)


def _plain_attn(s):
    c = s["case"]
    q = s["q"].unflatten(1, (c["kv_heads"], -1, c["size"]))
    pages = s["table"].clamp(min=0).long()
    # [request, page, head, position, dim] -> [request, head, positions, dim]
    k, v = (p[pages].transpose(1, 2).flatten(2, 3) for p in (s["kpool"], s["vpool"]))
    live = torch.arange(k.shape[2], device=k.device) < s["kv_len"][:, None]
    s["out"].copy_(_attend(q, k, v, live[:, None]).flatten(1))
    return s["out"]


def _plain_topk(s):
    c = s["case"]
    g, d, page, table = c["kv_heads"], c["size"], c["page"], s["table"].clamp(min=0).long()
    q = s["q"].unflatten(1, (g, -1, d))
    # the scores in 64 bits: which pages are taken must not depend on the order of a sum
    score = (q.double() @ s["means"][table].double().permute(0, 2, 3, 1)).amax(2)
    index = torch.arange(table.shape[1], device=q.device)
    total = ((s["kv_len"] + page - 1) // page)[:, None, None]
    kept = (index < c["sink"]) | (index >= total - c["window"])
    score = torch.where(kept, math.inf, score)
    score = torch.where(index < total, score, -math.inf)
    n = s["sel"].shape[2]
    best = torch.sort(score, dim=2, descending=True, stable=True).indices[..., :n]
    there = torch.arange(best.shape[2], device=q.device) < total
    best = torch.where(there, best, table.shape[1]).sort(2).values
    s["sel"].fill_(-1)
    s["sel"][..., :best.shape[2]] = torch.where(there, best, -1)
    best = torch.where(there, best, 0)
    mine = torch.gather(table[:, None].expand(-1, g, -1), 2, best)
    head = torch.arange(g, device=q.device)[:, None]
    k, v = (p[mine, head].flatten(2, 3) for p in (s["kpool"], s["vpool"]))
    at = best[..., None] * page + torch.arange(page, device=q.device)
    live = (there[..., None] & (at < s["kv_len"][:, None, None, None])).flatten(2)
    s["out"].copy_(_attend(q, k, v, live).flatten(1))
    return [s["out"], s["sel"]]


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "plan":
        return _exact_plan(s)
    if case["op"] == "append":
        return _exact_append(s)
    return _exact_attn(s)


def _exact_plan(s):
    """Request by request, on the host."""
    page = s["case"]["page"]
    past, add = s["past"].tolist(), s["add"].tolist()
    table, ring = s["table"].tolist(), s["ring"].tolist()
    head, count = s["free"].tolist()
    n_pages, cap = len(ring), s["slots"].shape[0]
    left, room, taken, given = count, cap, 0, 0
    slots, pos, cu, kv_len, granted = [], [], [0], [], []
    for i, (p, a) in enumerate(zip(past, add)):
        have = _pages(p, page)
        if a == -1:
            for j in range(have):
                ring[(head + count + given) % n_pages] = table[i][j]
                given += 1
            kv_len.append(0)
            granted.append(1)
            cu.append(cu[-1])
            continue
        need = _pages(p + a, page) - have
        fits = p + a <= len(table[i]) * page
        if fits:
            left, room = left - need, room - a
        yes = fits and (need == 0 or left >= 0) and (a == 0 or room >= 0)
        if yes:
            for j in range(need):
                table[i][have + j] = ring[(head + taken) % n_pages]
                taken += 1
            for j in range(p, p + a):
                slots.append(table[i][j // page] * page + j % page)
                pos.append(j)
        granted.append(int(yes))
        kv_len.append(p + (a if yes else 0))
        cu.append(cu[-1] + (a if yes else 0))
    rest = cap - len(slots)
    return [_ints(table), _ints(ring), _ints(slots + [-1] * rest, torch.int64), _ints(pos + [0] * rest), _ints(cu),
            _ints(kv_len), _ints(granted), _ints([(head + taken) % n_pages, count - taken + given])]


def _exact_append(s):
    c = s["case"]
    h, g, d, page, rope = c["heads"], c["kv_heads"], c["size"], c["page"], c["rope"]
    z = torch.zeros((), dtype=torch.float64, device="cuda")

    def made(x, bias, w, heads, turned):
        y = (x.double() + (bias.double() if bias is not None else z)).view(-1, heads, d)
        if w is not None:
            over = y.flatten(1)[:, None] if c["norm"] == "full" else y
            y = y * (over.square().sum(-1, keepdim=True) / over.shape[-1] + EPS).rsqrt() * w.double().view(-1, d)
        if turned and rope:
            j = torch.arange(rope // 2, device="cuda", dtype=torch.float64)
            turn = torch.polar(torch.ones_like(j)[None],
                               s["pos"].double()[:, None] * torch.exp(j * (-2.0 / rope * math.log(ROPE_BASE))))
            w2 = torch.complex(y[..., :rope // 2].contiguous(), y[..., rope // 2:rope].contiguous()) * turn[:, None]
            y = torch.cat([w2.real, w2.imag, y[..., rope:]], -1)
        return y

    q, k = made(s["q"], s["bq"], s["q_norm"], h, True), made(s["k"], s["bk"], s["k_norm"], g, True)
    v = made(s["v"], s["bv"], None, g, False)
    out = [q.flatten(1)]
    rows = s["slots"]
    for pool, new in ((s["kpool"], k), (s["vpool"], v)):
        n_pages = pool.shape[0]
        flat = pool.double().transpose(1, 2).reshape(n_pages * page, g, d)
        flat[rows] = new
        out.append(flat.view(n_pages, page, g, d).transpose(1, 2))
    if s["means"] is not None:
        m = s["means"].double()
        # a mean is taken of the keys as the cache holds them
        kept = out[1].to(s["kpool"].dtype).double()
        m[s["filled"]] = kept[s["filled"]].sum(2) / page
        out.append(m)
    return out


def _exact_attn(s):
    c = s["case"]
    g, d, page = c["kv_heads"], c["size"], c["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    sel = torch.full_like(s["sel"], -1) if c["op"] == "topk" else None
    heads = torch.arange(g, device="cuda")
    for i, n in enumerate(s["lens"]):
        if n == 0:
            continue
        total = _pages(n, page)
        row = s["table"][i, :total].long()
        q = s["q"][i].double().view(g, -1, d)
        chosen = torch.arange(total, device="cuda").repeat(g, 1)
        if sel is not None:
            few, _ = _chosen(c, n)
            if few < total:
                score = torch.einsum("grd,pgd->gpr", q, s["means"][row].double()).max(-1).values
                score[:, :c["sink"]] = math.inf
                score[:, total - c["window"]:] = math.inf
                # the few best of each head, the lower page first among equals
                order = torch.argsort(-score, dim=1, stable=True)[:, :few]
                chosen = order.sort(1).values
            sel[i, :, :few] = chosen
        for r in range(g):
            at = (chosen[r][:, None] * page + torch.arange(page, device="cuda")).flatten()
            at = at[at < n]
            k = s["kpool"][row[at // page], heads[r], at % page].double()
            v = s["vpool"][row[at // page], heads[r], at % page].double()
            w = torch.einsum("rd,nd->rn", q[r], k) / math.sqrt(d)
            out[i].view(g, -1, d)[r] = torch.einsum("rn,nd->rd", torch.exp(w - torch.logsumexp(w, 1, keepdim=True)), v)
    return out if sel is None else [out, sel]
