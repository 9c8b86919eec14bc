"""Requests that share pages of the key-value pool, as they are measured: cases, inputs, one pass.

Four kinds of pass:

* ``shared``: one new token per request, where groups of requests share the
  pages of a long prefix;
* ``select``: a beam search's choice of the best continuations over beams
  and vocabulary;
* ``fork``: rows of a block table that continue other rows (beams reordered,
  requests split, cut back or ended) and the copies of unfinished pages in
  the layers' pools;
* ``compact``: the pages in use moved to the lowest numbers, in the tables
  and in the layers' pools.

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


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # latency: four beams of one request of the 16-head model after a short prompt
        dict(name="shared_beams", op="shared", groups=1, members=4, prefix=300, alone=0, own=24, heads=16, kv_heads=16,
             size=128, act=F32, kv=F16, page=16, tokens_first=False),
        # a batch of the 32 / 4-head model behind one system prompt, every request with some text of its own
        dict(name="shared_batch", op="shared", groups=1, members=64, prefix=8192, alone=0, own=500, heads=32,
             kv_heads=4, size=128, act=BF16, kv=BF16, page=64, tokens_first=False),
        # several prompts with their beams, requests of their own between them, small pages, positions before heads
        dict(name="shared_groups", op="shared", groups=9, members=7, prefix=3001, alone=5, own=777, heads=28,
             kv_heads=4, size=64, act=F16, kv=F16, page=8, tokens_first=True),
        # a very long document that a few requests ask about
        dict(name="shared_long", op="shared", groups=1, members=8, prefix=131072, alone=0, own=200, heads=32,
             kv_heads=4, size=128, act=F32, kv=F16, page=64, tokens_first=False),
        # the cache at the reference's width
        dict(name="shared_f32", op="shared", groups=2, members=6, prefix=4097, alone=1, own=100, heads=16, kv_heads=16,
             size=128, act=F32, kv=F32, page=32, tokens_first=False),
        # one request's four beams over the 16-head model's vocabulary
        dict(name="select_one", op="select", n_seq=1, beams=4, pick=4, vocab=50304, type=F32, first=False, done=0.0),
        # a batch of beam searches over the 32 / 4-head model's vocabulary, logits as the decoder leaves them
        dict(name="select_batch", op="select", n_seq=32, beams=8, pick=8, vocab=151936, type=F32, first=False,
             done=0.0),
        # an odd vocabulary in 16 bits, twice as many continuations as beams, some beams finished
        dict(name="select_odd", op="select", n_seq=13, beams=5, pick=10, vocab=32003, type=BF16, first=False, done=0.3),
        # a beam search's step: every request's beams reordered, unfinished pages copied in all 16 layers
        dict(name="fork_beams", op="fork", n_seq=8, beams=8, ctx=1000, page=16, layers=16, kv_heads=4, size=128,
             kv=F16, cut=0.0, end=0.0, tokens_first=False),
        # a server's step: requests split, cut back to an earlier position or ended
        dict(name="fork_mixed", op="fork", n_seq=512, beams=1, ctx=4001, page=64, layers=2, kv_heads=4, size=64,
             kv=BF16, cut=0.1, end=0.2, tokens_first=True),
        # a half-empty pool of a few requests
        dict(name="compact_few", op="compact", n_seq=6, ctx=700, page=32, layers=4, kv_heads=2, size=128, kv=F32,
             full=0.5, most=64, tokens_first=False),
        # a large pool, everything moved at once
        dict(name="compact_all", op="compact", n_seq=128, ctx=4096, page=64, layers=2, kv_heads=4, size=128, kv=BF16,
             full=0.6, most=4096, tokens_first=False),
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_once(rng):
    op = rng.choice(["shared", "shared", "shared", "select", "select", "fork", "compact"])
    if op == "select":
        beams = _log(rng, 1, 32)
        return dict(op=op, n_seq=_log(rng, 1, 64), beams=beams, pick=min(32, beams * rng.choice([1, 1, 2])),
                    vocab=_log(rng, 300, 160000), type=rng.choice([F32, F32, F16, BF16]), first=rng.random() < 0.2,
                    done=rng.choice([0.0, 0.0, rng.uniform(0.1, 0.6)]))
    size = rng.choice([64, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8, 16])
    case = dict(op=op, kv_heads=kv_heads, size=size, tokens_first=rng.random() < 0.5)
    if op == "shared":
        act, kv = rng.choice(PAIRS)
        case.update(groups=_log(rng, 1, 16), members=_log(rng, 1, 64), prefix=_log(rng, 40, 131072),
                    alone=rng.choice([0, 0, _log(rng, 1, 16)]), own=_log(rng, 1, 2000),
                    heads=kv_heads * rng.choice([1, 2, 3, 4, 5, 7, 8, 8, 12, 16]), act=act, kv=kv,
                    page=rng.choice([8, 16, 32, 64, 128]))
        return case
    case.update(layers=_log(rng, 1, 16), kv=rng.choice([F32, F16, BF16]), page=rng.choice([8, 16, 32, 64, 128]))
    if op == "fork":
        beams = rng.choice([1, 1, 2, 3, 4, 5, 8, 16])
        case.update(n_seq=max(1, _log(rng, 1, 512) // beams), beams=beams, ctx=_log(rng, 20, 8192),
                    cut=rng.choice([0.0, rng.uniform(0.0, 0.5)]), end=rng.choice([0.0, rng.uniform(0.0, 0.3)]))
    else:
        case.update(n_seq=_log(rng, 1, 256), ctx=_log(rng, 20, 8192), full=rng.uniform(0.2, 0.95),
                    most=_log(rng, 8, 8192))
    return case


def draw(rng):
    most = {}
    for c in listed():
        most[c["op"]] = max(most.get(c["op"], 0), work(c)["bytes"])
    while True:
        case = _draw_once(rng)
        # the cost of the plain form goes by the values it handles, however few bytes hold them
        if work(case)["bytes"] <= most[case["op"]] and _values(case) <= 600_000_000:
            return case


def _values(case):
    """Values that the plain form handles at once, about: of one of the gathered pools, of the logits, of the pools."""
    op = case["op"]
    if op == "select":
        return case["n_seq"] * case["beams"] * case["vocab"] * 4
    width = case["kv_heads"] * case["size"]
    if op == "shared":
        return len(_requests(case)[0]) * _table_width(case) * case["page"] * width
    return _pool_pages(case) * case["page"] * width * case["layers"] * 2


def _spread(n, most, least=1):
    """n whole numbers up to `most`, evenly spread, the largest among them."""
    golden = 0.6180339887498949
    return [max(least, int(round(most * ((i * golden) % 1.0)))) if i else most for i in range(n)]


def _pages(length, page):
    return -(-length // page)


def _requests(case):
    """Of a shared case: (own lengths, group sizes, shared lengths), requests of no group behind the groups."""
    sizes = [max(1, m) for m in _spread(case["groups"], case["members"])]
    shared = _spread(case["groups"], case["prefix"])
    lens = _spread(sum(sizes) + case["alone"], case["own"], 0)
    return lens, sizes, shared


def _lengths(case):
    """The rows' cached positions in a fork or compact case; rows of one request are beams of one length."""
    out = []
    for x in _spread(case["n_seq"], case["ctx"]):
        out += [x] * case.get("beams", 1)
    return out


def _table_width(case):
    if case["op"] == "shared":
        return _pages(case["prefix"] // case["page"] * case["page"] + case["own"], case["page"])
    return _pages(case["ctx"], case["page"])


def _common(case, length):
    """Pages that the beams of one request in a fork case hold together: all but the last few."""
    return max(0, length // case["page"] - 2)


def _pool_pages(case):
    """Pages of the pool: those in use and some more."""
    page = case["page"]
    if case["op"] == "shared":
        lens, _, shared = _requests(case)
        return sum(_pages(x, page) for x in lens) + sum(x // page for x in shared) + 16
    if case["op"] == "fork":
        beams = case["beams"]
        held = sum(_common(case, x) + beams * (_pages(x, page) - _common(case, x)) for x in _lengths(case)[::beams])
        return held + len(_lengths(case)) + 16
    held = sum(_pages(x, page) for x in _lengths(case))
    return int(held / case["full"]) + 16


def _moves(case):
    """Pages that a compact case moves, on average over the places that the pages in use may have."""
    held, n = sum(_pages(x, case["page"]) for x in _lengths(case)), _pool_pages(case)
    return min(case["most"], int(held * (n - held) / n))


def work(case):
    op = case["op"]
    if op == "select":
        rows, picked = case["n_seq"] * case["beams"], case["n_seq"] * case["pick"]
        return {"bytes": rows * (case["vocab"] * DTYPE[case["type"]].itemsize + 8) + picked * 16,
                "flops": 4 * rows * case["vocab"]}
    page, g, d = case["page"], case["kv_heads"], case["size"]
    c = DTYPE[case["kv"]].itemsize
    if op == "shared":
        lens, sizes, shared = _requests(case)
        a, h = DTYPE[case["act"]].itemsize, case["heads"]
        moved = len(lens) * (2 * h * d * a + 4) + 4 * (2 * len(sizes) + 1)
        flops, i = 0, 0
        for m, x in zip(sizes + [1] * case["alone"], shared + [0] * case["alone"]):
            x = x // page * page
            moved += x * 2 * g * d * c + x // page * 4
            for n in lens[i:i + m]:
                moved += n * 2 * g * d * c + _pages(n, page) * 4
                flops += 4 * (x + n) * h * d
            i += m
        return {"bytes": moved, "flops": flops}
    lens, n_pages = _lengths(case), _pool_pages(case)
    entries = sum(_pages(x, page) for x in lens)
    if op == "fork":
        # about: a row in e of a request's beams goes on in place, the others' unfinished pages are copied
        copied = sum(x % page for x in lens) * (0.37 if case["beams"] > 1 else 0.2)
        ints = 2 * entries + 2 * n_pages + 8 * len(lens)
        return {"bytes": int(4 * ints + copied * 4 * g * d * c * case["layers"]), "flops": entries}
    ints = 2 * entries + 3 * n_pages + 2 * case["most"] + len(lens)
    return {"bytes": 4 * ints + _moves(case) * page * 4 * g * d * c * case["layers"], "flops": entries + n_pages}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype).cuda()


def _zeros(*shape, dtype=torch.int32):
    return torch.zeros(*shape, dtype=dtype, device="cuda")


def _pool(case, n_pages, gen):
    """A pool seen as [page, head, position, dim], whichever of heads and positions lies outside."""
    g, p, d = case["kv_heads"], case["page"], case["size"]
    dtype = DTYPE[case["kv"]]
    if case["tokens_first"]:
        return torch.randn(n_pages, p, g, d, generator=gen, device="cuda", dtype=dtype).transpose(1, 2)
    return torch.randn(n_pages, g, p, d, generator=gen, device="cuda", dtype=dtype)


def _handle(case, k, v):
    import vireo_b200
    return vireo_b200.PagedKV(k, v, case.get("heads", case["kv_heads"]), DTYPE[case.get("act", case["kv"])])


def prepare(case, seed):
    rng = random.Random(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    {"shared": _prepare_shared, "select": _prepare_select, "fork": _prepare_fork,
     "compact": _prepare_compact}[case["op"]](case, rng, gen, state)
    if own and case["op"] == "shared":
        state["kv"] = _handle(case, state["kpool"], state["vpool"])
    elif own and case["op"] != "select":
        state["kv"] = [_handle(case, k, v) for k, v in state["pools"]]
    return state


def _prepare_shared(case, rng, gen, state):
    lens, sizes, shared = _requests(case)
    page, n_pages, width = case["page"], _pool_pages(case), _table_width(case)
    rng.shuffle(lens)
    ids = list(range(n_pages))
    rng.shuffle(ids)
    rows, total, at, used = [], [], 0, 0
    for m, x in zip(sizes + [1] * case["alone"], shared + [0] * case["alone"]):
        first = ids[used:used + x // page]
        used += len(first)
        for n in lens[at:at + m]:
            k = _pages(n, page)
            rows.append(first + ids[used:used + k])
            total.append(len(first) * page + n)
            used += k
        at += m
    cu = [0]
    for m in sizes:
        cu.append(cu[-1] + m)
    kpool, vpool = _pool(case, n_pages, gen), _pool(case, n_pages, gen)
    # keys of one page resemble one another, as neighbouring tokens' do
    kpool.mul_(0.8).add_(torch.randn(n_pages, case["kv_heads"], 1, case["size"], generator=gen, device="cuda",
                                     dtype=kpool.dtype) * 0.6)
    act, w = DTYPE[case["act"]], case["heads"] * case["size"]
    state.update(kpool=kpool, vpool=vpool, table=_ints([r + [-1] * (width - len(r)) for r in rows]), lens=total,
                 kv_len=_ints(total), cu=_ints(cu), shared=_ints(shared),
                 q=torch.randn(len(rows), w, generator=gen, device="cuda").to(act),
                 out=torch.zeros(len(rows), w, device="cuda", dtype=act))


def _prepare_select(case, rng, gen, state):
    n, b, k, vocab = case["n_seq"], case["beams"], case["pick"], case["vocab"]
    logits = torch.randn(n * b, vocab, generator=gen, device="cuda") * 2.0
    # a few tokens stand out, as after training
    likely = torch.randint(0, vocab, (n * b, 12), generator=gen, device="cuda")
    logits.scatter_add_(1, likely, torch.rand(n * b, 12, generator=gen, device="cuda") * 12.0)
    score = -torch.rand(n * b, generator=gen, device="cuda") * 6.0 - 20.0
    if case["first"]:  # a search begins with one beam
        score = torch.where(torch.arange(n * b, device="cuda") % b == 0, 0.0, -math.inf)
    done = (torch.rand(n * b, generator=gen, device="cuda") < case["done"]).int() if case["done"] else None
    state.update(logits=logits.to(DTYPE[case["type"]]), score=score.float(), done=done,
                 score_out=_zeros(n, k, dtype=torch.float32), token=_zeros(n, k), parent=_zeros(n, k),
                 done_out=_zeros(n, k))


def _prepare_fork(case, rng, gen, state):
    page, beams, n_pages, width = case["page"], case["beams"], _pool_pages(case), _table_width(case)
    lens = _lengths(case)
    n = len(lens)
    ids = list(range(n_pages))
    rng.shuffle(ids)
    rows, shares, used = [], [0] * n_pages, 0
    for i in range(0, n, beams):  # beams of one request hold its first pages together
        first = ids[used:used + _common(case, lens[i])]
        used += len(first)
        for p in first:
            shares[p] = beams - 1
        for _ in range(beams):
            k = _pages(lens[i], page) - len(first)
            rows.append(first + ids[used:used + k])
            used += k
    free, head = ids[used:], rng.randrange(n_pages)
    ring = [-1] * n_pages
    for i, p in enumerate(free):
        ring[(head + i) % n_pages] = p
    parent, keep = [], []
    for i in range(n):
        s = i - i % beams
        # requests of one row: one in five is split in place of another
        p = s + rng.randrange(beams) if beams > 1 else (rng.randrange(n) if rng.random() < 0.2 else i)
        parent.append(-1 if rng.random() < case["end"] else p)
        keep.append(rng.randrange(0, lens[p] + 1) if rng.random() < case["cut"] else -1)
    state.update(kv_len=_ints(lens), table=_ints([r + [-1] * (width - len(r)) for r in rows]), parent=_ints(parent),
                 keep=_ints(keep) if case["cut"] else None, shares=_ints(shares), ring=_ints(ring),
                 free=_ints([head, len(free)]), table_out=_zeros(n, width) - 1, kv_len_out=_zeros(n),
                 granted=_zeros(n), shares_out=_zeros(n_pages), free_out=_zeros(2), src=_zeros(n), dst=_zeros(n),
                 rows=_zeros(n), pools=[(_pool(case, n_pages, gen), _pool(case, n_pages, gen))
                                        for _ in range(case["layers"])])


def _prepare_compact(case, rng, gen, state):
    page, n_pages, width = case["page"], _pool_pages(case), _table_width(case)
    lens = _lengths(case)
    ids = list(range(n_pages))
    rng.shuffle(ids)
    rows, shares, used = [], [0] * n_pages, 0
    for i, x in enumerate(lens):
        k = _pages(x, page)
        rows.append(ids[used:used + k])
        used += k
        if i % 4 == 3:  # one in four begins with pages of the one before it
            both = min(k, len(rows[i - 1])) // 2
            rows[i][:both] = rows[i - 1][:both]
            for p in rows[i][:both]:
                shares[p] += 1
    most = min(case["most"], n_pages // 2 + 1)
    state.update(kv_len=_ints(lens), table=_ints([r + [-1] * (width - len(r)) for r in rows]), shares=_ints(shares),
                 ring=_zeros(n_pages) - 1, table_out=_zeros(len(lens), width) - 1, shares_out=_zeros(n_pages),
                 free_out=_zeros(2), src=_zeros(most), dst=_zeros(most),
                 pools=[(_pool(case, n_pages, gen), _pool(case, n_pages, gen)) for _ in range(case["layers"])])


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return _own(op, state)
    return {"shared": _plain_shared, "select": _plain_select, "fork": _plain_fork, "compact": _plain_compact}[op](state)


def _select_outputs(s):
    return [s[n] for n in ("score_out", "token", "parent", "done_out")]


def _fork_outputs(s):
    return [s[n] for n in ("table_out", "kv_len_out", "granted", "shares_out", "ring", "free_out", "src", "dst",
                           "rows")] + [p for pools in s["pools"] for p in pools]


def _compact_outputs(s):
    return [s[n] for n in ("table_out", "shares_out", "ring", "free_out", "src", "dst")] + [
        p for pools in s["pools"] for p in pools]


def _own(op, s):
    c = s["case"]
    if op == "shared":
        s["kv"].attn_shared(s["q"], s["table"], s["kv_len"], s["cu"], s["shared"], s["out"])
        return s["out"]
    import vireo_b200
    if op == "select":
        vireo_b200.beam_select(s["logits"], s["score"], c["beams"], score_out=s["score_out"], token=s["token"],
                               parent=s["parent"], done=s["done"], done_out=s["done_out"], end_token=2)
        return _select_outputs(s)
    if op == "fork":
        vireo_b200.kv_fork(s["kv_len"], s["table"], s["parent"], s["shares"], s["ring"], s["free"], c["page"],
                           keep=s["keep"], table_out=s["table_out"], kv_len_out=s["kv_len_out"], granted=s["granted"],
                           shares_out=s["shares_out"], state_out=s["free_out"], src=s["src"], dst=s["dst"],
                           rows=s["rows"])
        vireo_b200.kv_copy(s["kv"], s["src"], s["dst"], rows=s["rows"])
        return _fork_outputs(s)
    vireo_b200.kv_compact(s["kv_len"], s["table"], s["ring"], c["page"], shares=s["shares"], table_out=s["table_out"],
                          shares_out=s["shares_out"], state_out=s["free_out"], src=s["src"], dst=s["dst"])
    vireo_b200.kv_copy(s["kv"], s["src"], s["dst"])
    return _compact_outputs(s)


def _plain_shared(s):
    c = s["case"]
    q = s["q"].float().unflatten(1, (c["kv_heads"], -1, c["size"]))
    pages = s["table"].clamp(min=0).long()
    # [request, page, head, position, dim] -> [request, head, positions, dim]
    k, v = (p[pages].transpose(1, 2).flatten(2, 3).float() for p in (s["kpool"], s["vpool"]))
    live = (torch.arange(k.shape[2], device=k.device) < s["kv_len"][:, None])[:, None, None]
    w = q @ k.transpose(2, 3) * (1.0 / math.sqrt(c["size"]))
    w = torch.where(live, w, -math.inf)
    w = torch.where(live, torch.exp(w - w.amax(-1, keepdim=True)), 0.0)
    total = w.sum(-1, keepdim=True)
    s["out"].copy_(torch.where(total > 0, w @ v / total, 0.0).flatten(1))
    return s["out"]


def _plain_select(s):
    c = s["case"]
    b, k, vocab = c["beams"], c["pick"], c["vocab"]
    # in 64 bits: two beams' totals may lie near one another
    x, score = s["logits"].double(), s["score"].double()[:, None]
    top = x.amax(1, keepdim=True)
    total = score + x - (top + torch.log(torch.exp(x - top).sum(1, keepdim=True)))
    if s["done"] is not None:
        done = s["done"][:, None] != 0
        ends = torch.arange(vocab, device=x.device) == 2
        total = torch.where(done, torch.where(ends, score, -math.inf), total)
    total = torch.where(torch.isfinite(total), total, -math.inf).view(c["n_seq"], b * vocab)
    total, at = torch.sort(total, dim=1, descending=True, stable=True)
    total, at = total[:, :k], at[:, :k]
    there = total > -math.inf
    parent = torch.arange(c["n_seq"], device=x.device)[:, None] * b + at // vocab
    token = torch.where(there, at % vocab, -1)
    s["score_out"].copy_(total)
    s["token"].copy_(token)
    s["parent"].copy_(torch.where(there, parent, -1))
    s["done_out"].copy_((token == 2) | (token < 0))
    return _select_outputs(s)


def _move(s, src, dst, rows):
    """Positions 0 .. rows - 1 of pages src to pages dst, where src is one, in every layer."""
    page = s["case"]["page"]
    # a pair that is none does what the first that is one does, or copies nothing of page 0 to itself
    pair = torch.where(src >= 0, torch.arange(len(src), device=src.device), (src >= 0).int().argmax())
    src, dst, rows = src.long()[pair], dst.long()[pair], rows[pair]
    rows = torch.where(src >= 0, rows, 0)
    src, dst = src.clamp(min=0), dst.clamp(min=0)
    live = (torch.arange(page, device=src.device) < rows[:, None])[:, None, :, None]
    for pools in s["pools"]:
        for p in pools:
            p[dst] = torch.where(live, p[src], p[dst])


def _plain_fork(s):
    page, dev = s["case"]["page"], s["table"].device
    table, kv_len, ring, shares = s["table"].long(), s["kv_len"].long(), s["ring"], s["shares"].long()
    n, width, n_pages = table.shape[0], table.shape[1], ring.shape[0]
    head, count = s["free"][0].long(), s["free"][1].long()
    parent = s["parent"].long()
    there = parent >= 0
    p = parent.clamp(min=0)
    keep = s["keep"].long() if s["keep"] is not None else torch.full_like(parent, -1)
    want = torch.where(there, torch.where(keep < 0, kv_len[p], torch.minimum(keep, kv_len[p])), 0)
    full, tail = want // page, want % page
    # who else of the parent's rows reaches the unfinished page, and who has all of it
    other = (parent[:, None] == parent[None]) & there[:, None]
    reach = other & (want[None] > (full * page)[:, None])
    whole = other & (want[None] >= ((full + 1) * page)[:, None])
    index = torch.arange(n, device=dev)
    earlier = (reach & (index[None] < index[:, None])).any(1)
    last = table[p].gather(1, full.clamp(max=width - 1)[:, None])[:, 0]
    stays = (tail > 0) & (shares[last.clamp(min=0)] == 0) & ~earlier & ~whole.any(1)
    need = (tail > 0) & ~stays
    rank = need.long().cumsum(0) - 1
    granted = ~need | (rank < count)
    fresh = ring.long()[(head + rank.clamp(min=0)) % n_pages]
    copied = need & granted
    held = torch.where(granted, full + (tail > 0).long(), 0)
    taken = torch.where(granted, full + stays.long(), 0)  # of the parent's own pages
    col = torch.arange(width, device=dev)
    rows = torch.where(copied[:, None] & (col == full[:, None]), fresh[:, None], table[p])
    s["table_out"].copy_(torch.where(col < held[:, None], rows, s["table_out"]))
    # holders: one less for every old entry, one more for every new one
    had = col < ((kv_len + page - 1) // page)[:, None]
    more = shares.new_zeros(n_pages + 1)
    more.index_add_(0, torch.where(had, table, n_pages).flatten(), -torch.ones_like(table).flatten())
    mine = col < taken[:, None]
    more.index_add_(0, torch.where(mine, table[p], n_pages).flatten(), torch.ones_like(table).flatten())
    now = shares + more[:n_pages]
    gone = now < 0
    back = gone.long().cumsum(0) - 1
    at = torch.where(gone, (head + count + back) % n_pages, n_pages)
    ring.copy_(torch.cat([ring, ring[:1]]).scatter(0, at, torch.arange(n_pages, device=dev, dtype=ring.dtype))[:n_pages])
    s["shares_out"].copy_(now.clamp(min=0))
    used = copied.long().sum()
    s["free_out"].copy_(torch.stack([(head + used) % n_pages, count - used + gone.long().sum()]))
    s["kv_len_out"].copy_(torch.where(granted, want, 0))
    s["granted"].copy_(granted)
    s["src"].copy_(torch.where(copied, last, -1))
    s["dst"].copy_(torch.where(copied, fresh, -1))
    s["rows"].copy_(torch.where(copied, tail, 0))
    _move(s, s["src"], s["dst"], s["rows"])
    return _fork_outputs(s)


def _plain_compact(s):
    page, dev, most = s["case"]["page"], s["table"].device, s["src"].shape[0]
    table, n_pages = s["table"].long(), s["ring"].shape[0]
    col = torch.arange(table.shape[1], device=dev)
    held = col < ((s["kv_len"].long() + page - 1) // page)[:, None]
    used = torch.zeros(n_pages + 1, dtype=torch.bool, device=dev)
    used = used.scatter(0, torch.where(held, table, n_pages).flatten(), True)[:n_pages]
    ids = torch.arange(n_pages, device=dev)
    total = used.long().sum()
    up, down = used.long().cumsum(0) - 1, (~used).long().cumsum(0) - 1
    # the highest pages in use, at most so many, of those that lie behind the first `total`
    late = (used & (ids >= total)).long().sum()
    moved = late.clamp(max=most)
    goes = used & (ids >= total) & (up >= total - moved)
    which = up - (total - moved)
    free = torch.full((n_pages + 1,), -1, dtype=torch.long, device=dev)
    free = free.scatter(0, torch.where(used, n_pages, down), ids)[:n_pages]  # by rank
    to = torch.where(goes, free[which.clamp(min=0)], ids)
    pad = torch.full((most + 1,), -1, dtype=torch.long, device=dev)
    src = pad.scatter(0, torch.where(goes, which, most), ids)[:most]
    slot = torch.arange(most, device=dev)
    s["src"].copy_(torch.where(slot < moved, src, -1))
    s["dst"].copy_(torch.where(slot < moved, free[slot.clamp(max=n_pages - 1)], -1))
    s["table_out"].copy_(torch.where(held, to[table.clamp(min=0)], s["table_out"].long()))
    goes_to = torch.where(goes, to, n_pages)
    shares = torch.where(goes, 0, s["shares"])
    s["shares_out"].copy_(torch.cat([shares, shares[:1]]).scatter(0, goes_to, s["shares"])[:n_pages])
    after = used & ~goes
    after = torch.cat([after, after[:1]]).scatter(0, goes_to, True)[:n_pages]
    left = (~after).long().cumsum(0) - 1
    ring = torch.cat([s["ring"], s["ring"][:1]]).scatter(0, torch.where(after, n_pages, left), ids.to(s["ring"].dtype))
    s["ring"].copy_(ring[:n_pages])
    s["free_out"].copy_(torch.stack([total * 0, n_pages - total]))
    _move(s, s["src"], s["dst"], torch.full_like(s["src"], page))
    return _compact_outputs(s)


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"shared": _exact_shared, "select": _exact_select, "fork": _exact_fork,
            "compact": _exact_compact}[case["op"]](s)


def _exact_shared(s):
    """Request by request."""
    c = s["case"]
    g, d, page = c["kv_heads"], c["size"], c["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for i, n in enumerate(s["lens"]):
        if n == 0:
            continue
        at = torch.arange(n, device="cuda")
        row = s["table"][i].long()[at // page]
        q = s["q"][i].double().view(g, -1, d)
        for h in range(g):
            w = torch.einsum("rd,nd->rn", q[h], s["kpool"][row, h, at % page].double()) / math.sqrt(d)
            w = torch.exp(w - torch.logsumexp(w, 1, keepdim=True))
            out[i].view(g, -1, d)[h] = torch.einsum("rn,nd->rd", w, s["vpool"][row, h, at % page].double())
    return out


def _exact_select(s):
    """Request by request: every beam's best tokens, then the best of those."""
    c = s["case"]
    b, k, vocab = c["beams"], c["pick"], c["vocab"]
    score, token, parent, done = [], [], [], []
    for i in range(c["n_seq"]):
        found = []
        for r in range(i * b, i * b + b):
            so_far = s["score"][r].item()
            if so_far == -math.inf:
                continue
            if s["done"] is not None and s["done"][r].item():
                found.append((-so_far, r, 2))
                continue
            x = s["logits"][r].double()
            lse = torch.logsumexp(x, 0).item()
            # all that reach the k-th best, so that equal ones are all there
            ids = torch.nonzero(x >= torch.topk(x, min(k, vocab)).values[-1])[:, 0].tolist()
            found += [(-(so_far + v - lse), r, t) for t, v in zip(ids, x[ids].tolist())]
        found = sorted(found)[:k]
        rest = k - len(found)
        score.append([-f[0] for f in found] + [-math.inf] * rest)
        parent.append([f[1] for f in found] + [-1] * rest)
        token.append([f[2] for f in found] + [-1] * rest)
        done.append([int(f[2] == 2) for f in found] + [1] * rest)
    return [_ints(score, torch.float64), _ints(token), _ints(parent), _ints(done)]


def _exact_fork(s):
    """Row by row, on the host."""
    page = s["case"]["page"]
    table, kv_len, parent = s["table"].tolist(), s["kv_len"].tolist(), s["parent"].tolist()
    keep = s["keep"].tolist() if s["keep"] is not None else [-1] * len(parent)
    shares, ring, (head, count) = s["shares"].tolist(), s["ring"].tolist(), s["free"].tolist()
    new, n_pages = s["table_out"].tolist(), len(s["ring"])
    children = {}
    for i, p in enumerate(parent):
        if p >= 0:
            children.setdefault(p, []).append((i, kv_len[p] if keep[i] < 0 else min(keep[i], kv_len[p])))
    lens, granted, src, dst, rows, holders = [0] * len(parent), [1] * len(parent), [], [], [], list(shares)
    for i, p in enumerate(table):
        for j in range(_pages(kv_len[i], page)):
            holders[p[j]] -= 1
    used = 0
    for i, p in enumerate(parent):
        pair = (-1, -1, 0)
        if p >= 0:
            want = dict(children[p])[i]
            whole, tail = divmod(want, page)
            row = table[p][:whole]
            if tail:
                last = table[p][whole]
                near = [(c, w) for c, w in children[p] if w > whole * page]
                if shares[last] == 0 and near[0][0] == i and all(w < (whole + 1) * page for _, w in near):
                    row = row + [last]
                elif used < count:
                    pair = (last, ring[(head + used) % n_pages], tail)
                    used += 1
                else:
                    granted[i] = 0
            if granted[i]:
                for q in row:
                    holders[q] += 1
                lens[i] = want
                row = row + ([pair[1]] if pair[2] else [])
                new[i][:len(row)] = row
        src.append(pair[0])
        dst.append(pair[1])
        rows.append(pair[2])
    gone = [q for q in range(n_pages) if holders[q] < 0]
    for j, q in enumerate(gone):
        ring[(head + count + j) % n_pages] = q
    return [_ints(new), _ints(lens), _ints(granted), _ints([max(h, 0) for h in holders]), _ints(ring),
            _ints([(head + used) % n_pages, count - used + len(gone)]), _ints(src), _ints(dst), _ints(rows)] + [
                None for pools in s["pools"] for _ in pools]


def _exact_compact(s):
    """Page by page, on the host."""
    page, most, n_pages = s["case"]["page"], len(s["src"]), len(s["ring"])
    table, kv_len, shares, new = (s[n].tolist() for n in ("table", "kv_len", "shares", "table_out"))
    used = {q for row, n in zip(table, kv_len) for q in row[:_pages(n, page)]}
    behind = sorted(q for q in used if q >= len(used))
    src = behind[len(behind) - min(most, len(behind)):]
    free = [q for q in range(n_pages) if q not in used]
    dst = free[:len(src)]
    to = dict(zip(src, dst))
    for row, out, n in zip(table, new, kv_len):
        for j in range(_pages(n, page)):
            out[j] = to.get(row[j], row[j])
    for a, b in to.items():
        shares[a], shares[b] = 0, shares[a]
    after = {to.get(q, q) for q in used}
    ring = [q for q in range(n_pages) if q not in after]
    pad = [-1] * (most - len(src))
    return [_ints(new), _ints(shares), _ints(ring + s["ring"].tolist()[len(ring):]), _ints([0, len(ring)]),
            _ints(src + pad), _ints(dst + pad)] + [None for pools in s["pools"] for _ in pools]
