"""The paged key/value cache and its attention, as work to be measured: the
write of a step's keys and values into the cache's pages (with the per-head
norm and rotation before it), the attention of new tokens over the pages (a
prompt chunk, a ragged batch of chunks, single tokens), and the page
operations between steps (grow, fork, free, compact).

Every operator is here twice: in its plain form (elementary torch operations
in 32 bits, rounded once at the end), and as the calls a user of the library
makes (`own`)."""
import math
import random
import sys
from pathlib import Path

import torch

own = False

EPS, ROPE_BASE = 1e-6, 1e6
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


# --- the cases ---------------------------------------------------------------


def listed():
    attend = dict(op="attend", causal=True, window=0, ragged=False)
    append = dict(op="append", norm=True, neox=True)
    return [
        # the whole-model prefill's last full chunk of 2,048 tokens (32 query heads on 8, head size 128)
        dict(attend, name="chunk 2048 over 8192", type="bf16", seqs=1, q=2048, kv=8192, heads=32, kv_heads=8, d=128,
             page=64),
        # the same chunk deep in a long context: the largest work
        dict(attend, name="chunk 2048 over 32768", type="bf16", seqs=1, q=2048, kv=32768, heads=32, kv_heads=8,
             d=128, page=64),
        # a 27B-class layer's first chunk (24 query heads on 4, head size 256), f16 cache
        dict(attend, name="chunk 2048 of 2048, d 256", type="f16", seqs=1, q=2048, kv=2048, heads=24, kv_heads=4,
             d=256, page=64),
        # several users' short prompts in one ragged batch, small heads, small pages
        dict(attend, name="ragged prompts, d 64", type="bf16", seqs=6, q=700, kv=1500, heads=32, kv_heads=8, d=64,
             page=16, ragged=True),
        # the first tokens of an answer: one sequence, one token, a short cache (latency)
        dict(attend, name="token over 1000", type="bf16", seqs=1, q=1, kv=1000, heads=32, kv_heads=8, d=128, page=64),
        # a serving step: many sequences of many lengths, one token each
        dict(attend, name="32 tokens, ragged to 8192", type="f16", seqs=32, q=1, kv=8192, heads=32, kv_heads=8, d=128,
             page=16, ragged=True),
        # one token over a very long context
        dict(attend, name="token over 131072", type="bf16", seqs=1, q=1, kv=131072, heads=32, kv_heads=8, d=128,
             page=64),
        # a serving step's new keys and values: one token of each of 32 sequences
        dict(append, name="append 32 tokens", type="bf16", seqs=32, q=1, kv=4000, heads=32, kv_heads=8, d=128,
             rot=128, page=16),
        # a prompt chunk's
        dict(append, name="append 2048", type="bf16", seqs=1, q=2048, kv=8192, heads=32, kv_heads=8, d=128, rot=128,
             page=64),
        # a prompt shared by several continuations: whole pages shared, part pages copied in every layer
        dict(op="fork", name="fork 8", type="bf16", seqs=24, n=8, kv=3000, layers=36, kv_heads=8, d=128, page=16,
             pages=5000),
        # a fragmented pool after many sequences have ended
        dict(op="compact", name="compact 512 pages", type="bf16", seqs=24, n=10, kv=2000, layers=12, kv_heads=8,
             d=128, page=64, pages=512),
        # a serving step's bookkeeping: new pages for the sequences that cross into one
        dict(op="grow", name="grow 32", type="bf16", seqs=48, n=32, kv=4000, layers=1, kv_heads=8, d=128, page=16,
             pages=13000),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    op = rng.choice(["attend"] * 5 + ["append"] * 2 + ["fork", "compact", "grow", "free"])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 8])
    group = rng.choice([1, 2, 3, 4, 4, 5, 6, 8])
    d = rng.choice([64, 128, 128, 256, 80, 96])
    c = dict(op=op, type=rng.choice(["bf16", "f16"]), kv_heads=kv_heads, d=d, page=rng.choice([16, 32, 64, 128]))
    if op == "attend":
        c |= dict(heads=kv_heads * group, causal=rng.random() < 0.85, ragged=rng.random() < 0.5)
        if rng.random() < 0.4:  # single tokens, or a few at a time
            c |= dict(seqs=_log(rng, 1, 64), q=rng.choice([1, 1, 1, 2, 5]))
            c["kv"] = max(c["q"], _log(rng, 1, min(131072, 500000 // c["seqs"])))
        else:
            c |= dict(seqs=rng.choice([1, 1, 2, 3, 7]), q=_log(rng, 17, 2048))
            # no more scores than the largest listed case has
            c["kv"] = c["q"] + _log(rng, 1, min(40000, max(2, (1 << 30) // (c["seqs"] * c["q"] * c["heads"]))))
        c["window"] = _log(rng, 8, 4096) if c["causal"] and rng.random() < 0.25 else 0
    elif op == "append":
        few = rng.random() < 0.5
        c |= dict(heads=kv_heads * group, seqs=_log(rng, 1, 64) if few else rng.choice([1, 2, 3]),
                  q=1 if few else _log(rng, 3, 4096), norm=rng.random() < 0.6, neox=rng.random() < 0.6)
        c |= dict(kv=c["q"] + _log(rng, 1, 4000), rot=rng.choice([d, d, d // 2]))
    else:
        seqs = _log(rng, 8, 64)
        c |= dict(seqs=seqs, n=rng.randint(1, seqs // 3), kv=_log(rng, 40, 4000), layers=rng.choice([1, 4, 12]))
        held = seqs * (c["kv"] // c["page"] + 2)
        c["pages"] = held + rng.randint(held // 8, held)
        while c["pages"] * c["page"] * kv_heads * d * c["layers"] > 1 << 29:
            c["layers"] = max(1, c["layers"] // 2)
            c["kv"] = max(40, c["kv"] // 2)
            held = seqs * (c["kv"] // c["page"] + 2)
            c["pages"] = held + held // 2
    return c


def _lengths(c):
    """[(new tokens, cached tokens with them)] of a case's sequences: the same
    for every seed, since the work goes by them."""
    if not c.get("ragged"):
        return [(c["q"], c["kv"])] * c["seqs"]
    r = random.Random(c["q"] * 1000003 + c["kv"] * 101 + c["seqs"])
    got = []
    for i in range(c["seqs"]):
        q = max(1, int(c["q"] * r.uniform(0.2, 1.0))) if i else c["q"]
        got.append((q, max(q, int(c["kv"] * r.uniform(0.05, 1.0))) if i else c["kv"]))
    return got


# --- inputs --------------------------------------------------------------------


def _pages_of(n, page):
    return -(-n // page)


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    return (_prepare_step if case["op"] in ("attend", "append") else _prepare_pages)(case, seed, g)


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=g, dtype=torch.float32).to(dtype)


def _prepare_step(c, seed, g):
    """A batch of sequences over one layer's cache, its pages in no order."""
    lens, page, dt = _lengths(c), c["page"], TYPES[c["type"]]
    T = sum(q for q, _ in lens)
    width = max(_pages_of(kv, page) for _, kv in lens)
    pages = sum(_pages_of(kv, page) for _, kv in lens) + 3
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    order = random.Random(seed).sample(range(pages), pages)
    table, at = [], 0
    for _, kv in lens:
        n = _pages_of(kv, page)
        table.append(order[at:at + n] + [-1] * (width - n))
        at += n
    starts = [0]
    for q, _ in lens:
        starts.append(starts[-1] + q)
    kv_heads, d, heads = c["kv_heads"], c["d"], c["heads"]
    pool = lambda: _randn(g, 1, pages, page, kv_heads, d, dtype=dt)  # noqa: E731
    s = dict(case=c, k=pool(), v=pool(), q_start=i32(starts), kv_len=i32([kv for _, kv in lens]), table=i32(table),
             max_q=max(q for q, _ in lens), max_kv=max(kv for _, kv in lens), T=T,
             err=torch.zeros(1, dtype=torch.int32, device="cuda"))
    if c["op"] == "attend":
        # normed and rotated queries: a spread of sharp and flat rows
        s["q"] = (_randn(g, T, heads, d) * (0.5 + torch.rand(T, heads, 1, device="cuda", generator=g))).to(dt)
        s["out"] = torch.zeros(T, heads, d, dtype=dt, device="cuda")
    else:
        s |= dict(q=_randn(g, T, heads, d) * 1.5, kn=_randn(g, T, kv_heads, d) * 1.5, vn=_randn(g, T, kv_heads, d),
                  q_out=torch.zeros(T, heads, d, dtype=dt, device="cuda"))
        w = lambda: torch.rand(d, device="cuda", generator=g) + 0.5  # noqa: E731
        s |= dict(q_norm=w() if c["norm"] else None, k_norm=w() if c["norm"] else None)
        pos = torch.cat([torch.arange(kv - q, kv, dtype=torch.float64) for q, kv in lens]).cuda()
        inv = ROPE_BASE ** (-torch.arange(0, c["rot"], 2, device="cuda", dtype=torch.float64) / c["rot"])
        ang = pos[:, None] * inv
        s["rope"] = torch.stack([ang.cos(), ang.sin()], -1).float().reshape(T, c["rot"])
    return s


def _prepare_pages(c, seed, g):
    """A pool in use: sequences of several lengths, one of them sharing its
    first pages with another, some ended, their pages free again."""
    r, page, pages, seqs, n = random.Random(seed), c["page"], c["pages"], c["seqs"], c["n"]
    width = _pages_of(c["kv"], page) + 1
    order = r.sample(range(pages), pages)
    ended = set(r.sample(range(2, seqs), n)) if c["op"] in ("fork", "compact") else set()
    table, lens, refs, at = [[-1] * width for _ in range(seqs)], [0] * seqs, [0] * pages, 0
    for s in range(seqs):
        if s in ended:
            at += r.randint(0, 3)  # holes where they were
            continue
        lens[s] = r.randint(max(1, c["kv"] // 2), c["kv"])
        shared = lens[0] // page if s == 1 else 0
        shared = min(shared, lens[s] // page)
        for j in range(_pages_of(lens[s], page)):
            if j < shared:
                table[s][j] = table[0][j]
            else:
                table[s][j] = order[at]
                at += 1
            refs[table[s][j]] += 1
    dt = TYPES[c["type"]]
    pool = lambda: torch.empty(c["layers"], pages, page, c["kv_heads"], c["d"], dtype=dt,  # noqa: E731
                               device="cuda").normal_(generator=g)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    s = dict(case=c, k=pool(), v=pool(), refs=i32(refs), table=i32(table), len=i32(lens),
             err=torch.zeros(1, dtype=torch.int32, device="cuda"))
    s |= dict(refs_out=torch.empty_like(s["refs"]), table_out=torch.empty_like(s["table"]),
              len_out=torch.empty_like(s["len"]))
    living = [x for x in range(seqs) if x not in ended]
    if c["op"] == "fork":
        dst = sorted(ended)
        s |= dict(src=i32([r.choice(living) for _ in dst]), dst=i32(dst))
    elif c["op"] != "compact":
        who = r.sample(living, n)
        s |= dict(seq=i32(who), add=i32([r.randint(1, page) for _ in who]))
    return s


# --- one pass ------------------------------------------------------------------


def run(state):
    return (_run_own if own else _run_plain)(state)


def _library():
    path = str(Path(__file__).resolve().parents[1] / "ggml-xdna_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import zest_b200
    return zest_b200


def _run_own(s):
    Z, c = _library(), s["case"]
    cache = Z.KvCache(s["k"], s["v"])
    if c["op"] in ("attend", "append"):
        batch = Z.KvBatch(s["q_start"], s["kv_len"], s["table"], T=s["T"], max_q=s["max_q"], max_kv=s["max_kv"])
        if c["op"] == "attend":
            return Z.kv_attend(cache, 0, batch, s["q"], causal=c["causal"], window=c["window"], out=s["out"],
                               err=s["err"])
        Z.kv_append(cache, 0, batch, s["kn"], s["vn"], q=s["q"], q_out=s["q_out"], k_norm=s["k_norm"],
                    q_norm=s["q_norm"], eps=EPS if c["norm"] else -1.0, rope=s["rope"], mode=Z.ROPE_NEOX if c["neox"] else Z.ROPE_NORMAL,
                    err=s["err"])
        return s["q_out"], s["k"], s["v"]
    tables = Z.KvTables(s["refs"], s["table"], s["len"])
    out = Z.KvTables(s["refs_out"], s["table_out"], s["len_out"])
    if c["op"] == "fork":
        Z.kv_fork(cache, tables, s["src"], s["dst"], out=out, err=s["err"])
    elif c["op"] == "compact":
        Z.kv_compact(cache, tables, out=out, err=s["err"])
    elif c["op"] == "grow":
        Z.kv_grow(cache, tables, s["seq"], s["add"], out=out, err=s["err"])
    else:
        Z.kv_free(cache, tables, s["seq"], out=out, err=s["err"])
    moved = (s["k"], s["v"]) if c["op"] in ("fork", "compact") else ()
    return s["refs_out"], s["table_out"], s["len_out"], *moved


def _run_plain(s):
    op = s["case"]["op"]
    if op == "attend":
        return _attend(s)
    if op == "append":
        return _append(s)
    return {"fork": _fork, "compact": _compact, "grow": _grow, "free": _free}[op](s)


def _slots(s):
    """(sequence, index among its new tokens) of each row of the batch."""
    row = torch.arange(s["T"], device="cuda")
    seq = torch.searchsorted(s["q_start"], row, right=True, out_int32=False) - 1
    return seq, row - s["q_start"][seq]


def _attend(s):
    c, page = s["case"], s["case"]["page"]
    seqs, width = s["table"].shape
    kv_heads, d, heads = c["kv_heads"], c["d"], c["heads"]
    new = s["q_start"].diff().long()
    seq, i = _slots(s)
    # the rows of each sequence side by side, the pages of each laid end to end
    q = torch.zeros(seqs, s["max_q"], heads, d, device="cuda")
    q[seq, i] = s["q"].float()
    q = q.view(seqs, s["max_q"], kv_heads, heads // kv_heads, d).permute(0, 2, 3, 1, 4)
    key = torch.arange(width * page, device="cuda")
    there = key < s["kv_len"].long()[:, None]
    k, v = (torch.where(there[..., None, None], x[0][s["table"].clamp(min=0).long()].flatten(1, 2).float(), 0.0)
            .permute(0, 2, 1, 3) for x in (s["k"], s["v"]))
    k, v = k[:, :, None], v[:, :, None]
    pos = (s["kv_len"].long() - new)[:, None] + torch.arange(s["max_q"], device="cuda")
    sees = there[:, None, :].expand(-1, s["max_q"], -1)
    if c["causal"]:
        sees = sees & (key <= pos[..., None])
    if c["window"]:
        sees = sees & (key > pos[..., None] - c["window"])
    score = torch.matmul(q * (1.0 / math.sqrt(d)), k.transpose(-1, -2))
    score.masked_fill_(~sees[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = score.sum(-1, keepdim=True)
    o = torch.matmul(score, v) / torch.where(total == 0.0, 1.0, total)
    o = o.permute(0, 3, 1, 2, 4).reshape(seqs, s["max_q"], heads, d)
    s["out"].copy_(o[seq, i])
    return s["out"]


def _turned(x, norm, rope, neox):
    """Per-head norm and rotation, in 32 bits."""
    if norm is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * norm
    rot = rope.shape[1]
    cs = rope.view(-1, 1, rot // 2, 2)
    cos, sin = cs[..., 0], cs[..., 1]
    head, rest = x[..., :rot], x[..., rot:]
    a, b = (head[..., :rot // 2], head[..., rot // 2:]) if neox else (head[..., 0::2], head[..., 1::2])
    a, b = a * cos - b * sin, a * sin + b * cos
    head = torch.cat([a, b], -1) if neox else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([head, rest], -1)


def _append(s):
    c, page = s["case"], s["case"]["page"]
    seq, i = _slots(s)
    pos = s["kv_len"].long()[seq] - s["q_start"].diff().long()[seq] + i
    at, slot = s["table"][seq, pos // page].long(), pos % page
    s["k"][0][at, slot] = _turned(s["kn"], s["k_norm"], s["rope"], c["neox"]).to(s["k"].dtype)
    s["v"][0][at, slot] = s["vn"].to(s["v"].dtype)
    s["q_out"].copy_(_turned(s["q"], s["q_norm"], s["rope"], c["neox"]))
    return s["q_out"], s["k"], s["v"]


def _free_pages(refs):
    """Every page's index, the free ones first, each kind in rising order."""
    return torch.argsort((refs != 0).int(), stable=True)


def _tables_out(s, refs, table, lens, moved=False):
    s["refs_out"].copy_(refs)
    s["table_out"].copy_(table)
    s["len_out"].copy_(lens)
    return s["refs_out"], s["table_out"], s["len_out"], *((s["k"], s["v"]) if moved else ())


def _grow(s):
    page, width = s["case"]["page"], s["table"].shape[1]
    who = s["seq"].long()
    lens = s["len"].index_add(0, who, s["add"])
    held, want = (-(-x[who].long() // page) for x in (s["len"], lens))
    first = torch.cumsum(want - held, 0) - (want - held)
    free = _free_pages(s["refs"])
    at = torch.arange(width, device="cuda")
    fresh = (at >= held[:, None]) & (at < want[:, None])
    pick = free[torch.where(fresh, first[:, None] + at - held[:, None], 0)]
    rows = torch.where(fresh, pick.int(), s["table"][who])
    refs = s["refs"].index_add(0, pick.flatten(), fresh.flatten().int())
    return _tables_out(s, refs, s["table"].index_copy(0, who, rows), lens)


def _free(s):
    who = s["seq"].long()
    rows = s["table"][who]
    refs = s["refs"].index_add(0, rows.clamp(min=0).flatten().long(), -(rows >= 0).flatten().int())
    return _tables_out(s, refs, s["table"].index_fill(0, who, -1), s["len"].index_fill(0, who, 0))


def _fork(s):
    page, width = s["case"]["page"], s["table"].shape[1]
    src, dst = s["src"].long(), s["dst"].long()
    length = s["len"][src]
    whole, part = length.long() // page, length.long() % page > 0
    at = torch.arange(width, device="cuda")
    shared, last = at < whole[:, None], (at == whole[:, None]) & part[:, None]
    fresh = _free_pages(s["refs"])[torch.cumsum(part.long(), 0) - part.long()]
    old = s["table"][src]
    rows = torch.where(shared, old, torch.where(last, fresh[:, None].int(), -1))
    refs = s["refs"].index_add(0, rows.clamp(min=0).flatten().long(), (rows >= 0).flatten().int())
    # a pair whose sequence ends with its page writes its first page onto itself
    first = old[:, 0].long()
    into = torch.where(part, fresh, first)
    since = torch.where(part, old.gather(1, whole.clamp(max=width - 1)[:, None])[:, 0].long(), first)
    for x in (s["k"], s["v"]):
        x[:, into] = x[:, since]
    return _tables_out(s, refs, s["table"].index_copy(0, dst, rows), s["len"].index_copy(0, dst, length), True)


def _compact(s):
    refs, pages = s["refs"], s["refs"].shape[0]
    at = torch.arange(pages, device="cuda")
    live = refs != 0
    count = live.sum()
    hole, high = ~live & (at < count), live & (at >= count)
    # the k-th live page above the count goes into the k-th hole below it
    holes, highs = (torch.argsort((~m).int(), stable=True) for m in (hole, high))
    n = hole.sum()
    k = torch.arange(pages, device="cuda")
    to = torch.scatter(at, 0, highs, torch.where(k < n, holes, highs))
    inverse = torch.scatter(at, 0, holes, torch.where(k < n, highs, holes))
    moved = torch.where(live & (to == at), refs, torch.where(hole, refs[inverse], 0))
    table = torch.where(s["table"] >= 0, to[s["table"].clamp(min=0).long()].int(), -1)
    n = int(n)  # as many pages as move
    for x in (s["k"], s["v"]):
        x[:, holes[:n]] = x[:, highs[:n]]
    return _tables_out(s, moved, table, s["len"], True)


# --- what a pass cannot do without ------------------------------------------------


def work(case):
    c = case
    if c["op"] in ("attend", "append"):
        lens, size = _lengths(c), 2
        T = sum(q for q, _ in lens)
        if c["op"] == "append":
            values = T * (c["heads"] + 2 * c["kv_heads"]) * c["d"]
            return {"bytes": values * 6 + T * c["rot"] * 4, "flops": values * (4 if c["norm"] else 1) + 3 * values}
        pairs = keys = 0
        for q, kv in lens:
            lo = 0
            if c["causal"]:
                for_row = lambda p: min(p + 1, c["window"]) if c["window"] else p + 1  # noqa: E731
                first = kv - q
                if c["window"]:
                    pairs += sum(for_row(p) for p in range(first, kv))
                    lo = max(0, first - c["window"] + 1)
                else:
                    pairs += q * (first + 1) + q * (q - 1) // 2
            else:
                pairs += q * kv
            keys += kv - lo
        return {"bytes": size * (2 * keys * c["kv_heads"] * c["d"] + 2 * T * c["heads"] * c["d"]),
                "flops": 4.0 * pairs * c["heads"] * c["d"]}
    page_bytes = 2 * c["layers"] * c["page"] * c["kv_heads"] * c["d"] * 2
    width = _pages_of(c["kv"], c["page"]) + 1
    tables = 2 * 4 * (c["pages"] + c["seqs"] * (width + 1))
    if c["op"] == "fork":
        moves = c["n"] * (c["page"] - 1) // c["page"]
    elif c["op"] == "compact":  # live pages above the count of live ones, for pages in random order
        live = min(c["pages"], (c["seqs"] - c["n"]) * (3 * c["kv"] // (4 * c["page"]) + 1))
        moves = live * (c["pages"] - live) // c["pages"]
    else:
        moves = 0
    return {"bytes": tables + 2 * moves * page_bytes, "flops": c["pages"]}


# --- the definitions, in 64 bits ---------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"attend": _exact_attend, "append": _exact_append}.get(case["op"], _exact_pages)(s)


def _laid_out(pool, row, kv, page):
    n = _pages_of(kv, page)
    return torch.cat([pool[0, p] for p in row[:n].tolist()])[:kv].double()


def _exact_attend(s):
    c = s["case"]
    starts, lens = s["q_start"].tolist(), s["kv_len"].tolist()
    if sum((b - a) * kv for a, b, kv in zip(starts, starts[1:], lens)) * c["heads"] > 1 << 32:
        return None
    out = torch.zeros(s["T"], c["heads"], c["d"], dtype=torch.float64, device="cuda")
    group = c["heads"] // c["kv_heads"]
    for x, kv in enumerate(lens):
        a, b = starts[x], starts[x + 1]
        k, v = (_laid_out(p, s["table"][x], kv, c["page"]) for p in (s["k"], s["v"]))
        pos = torch.arange(kv - (b - a), kv, device="cuda")[:, None]
        j = torch.arange(kv, device="cuda")[None]
        hidden = torch.zeros(b - a, kv, dtype=torch.bool, device="cuda")
        if c["causal"]:
            hidden |= j > pos
        if c["window"]:
            hidden |= j <= pos - c["window"]
        for h in range(c["heads"]):
            z = s["q"][a:b, h].double() @ k[:, h // group].T / math.sqrt(c["d"])
            z[hidden] = -math.inf
            out[a:b, h] = torch.softmax(z, -1).nan_to_num(0.0) @ v[:, h // group]
    return out


def _exact_append(s):
    c = s["case"]
    cs = s["rope"].double()

    def turned(x, w):
        x = x.double()
        if w is not None:
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / c["d"] + EPS) * w.double()
        y = x.clone()
        for p in range(c["rot"] // 2):
            a, b = (p, p + c["rot"] // 2) if c["neox"] else (2 * p, 2 * p + 1)
            co, si = cs[:, 2 * p, None], cs[:, 2 * p + 1, None]
            y[..., a] = x[..., a] * co - x[..., b] * si
            y[..., b] = x[..., a] * si + x[..., b] * co
        return y

    k, v = s["k"].double(), s["v"].double()
    kn, vn = turned(s["kn"], s["k_norm"]), s["vn"].double()
    starts, lens, page = s["q_start"].tolist(), s["kv_len"].tolist(), c["page"]
    for x, kv in enumerate(lens):
        row, n = s["table"][x].tolist(), starts[x + 1] - starts[x]
        p = kv - n
        while p < kv:  # the new tokens of one page at a time
            m, t = min(page - p % page, kv - p), starts[x] + p - (kv - n)
            k[0, row[p // page], p % page:p % page + m] = kn[t:t + m]
            v[0, row[p // page], p % page:p % page + m] = vn[t:t + m]
            p += m
    return turned(s["q"], s["q_norm"]), k, v


def _exact_pages(s):
    """The tables by the definition, page by page on the host."""
    c, page = s["case"], s["case"]["page"]
    refs, table, lens = s["refs"].tolist(), s["table"].tolist(), s["len"].tolist()
    moves = []
    take = lambda: next(p for p, r in enumerate(refs) if r == 0)  # noqa: E731
    if c["op"] == "grow":
        for x, n in zip(s["seq"].tolist(), s["add"].tolist()):
            for j in range(_pages_of(lens[x], page), _pages_of(lens[x] + n, page)):
                table[x][j] = take()
                refs[table[x][j]] = 1
            lens[x] += n
    elif c["op"] == "free":
        for x in s["seq"].tolist():
            for p in table[x]:
                if p >= 0:
                    refs[p] -= 1
            table[x], lens[x] = [-1] * len(table[x]), 0
    elif c["op"] == "fork":
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            for j in range(_pages_of(lens[a], page)):
                if (j + 1) * page <= lens[a]:
                    table[b][j] = table[a][j]
                else:
                    table[b][j] = take()
                    moves.append((table[a][j], table[b][j]))
                refs[table[b][j]] += 1
            lens[b] = lens[a]
    else:
        live = sum(r > 0 for r in refs)
        high = [p for p in range(live, len(refs)) if refs[p]]
        for a, b in zip(high, [p for p in range(live) if not refs[p]]):
            moves.append((a, b))
            refs[a], refs[b] = 0, refs[a]
        to = dict(moves)
        table = [[to.get(p, p) for p in row] for row in table]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    pools = ()
    if c["op"] in ("fork", "compact"):
        pools = s["k"].double(), s["v"].double()
        for a, b in moves:
            for x in pools:
                x[:, b] = x[:, a]
    return i32(refs), i32(table), i32(lens), *pools
