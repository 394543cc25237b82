"""The paged cache's own operations against their definitions: what
zest_kv_append writes (64 bits; a value is rounded once to the cache's type,
half a step, and the norm and rotation before it are f32: a d-term sum, a
square root, a division and four products, below 2^-19 of the row's largest
value), the page tables against the host's model number by number, and a
serving loop that runs all of it with the attention."""
import math
import random

import pytest
import torch

import zest_b200 as Z
from kv_util import Pages, attention, turned

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def rope_table(pos, n_dims, base=1e6):
    ang = torch.tensor(pos, dtype=torch.float64)[:, None] * base ** (
        -torch.arange(0, n_dims, 2, dtype=torch.float64) / n_dims)
    return torch.stack([ang.cos(), ang.sin()], -1).float().reshape(len(pos), n_dims).cuda()


def near(got, want, dt):
    """Rounded once to dt from f32 that is within 2^-19 of the row's largest value."""
    want = want.reshape(got.shape)
    tol = torch.finfo(dt).eps / 2 * want.abs() + 2.0 ** -19 * want.abs().amax(-1, keepdim=True)
    if dt == HF:
        tol += 2.0 ** -25
    return bool(((got.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("dt,d,heads,kv_heads,page,lens,eps,weights,n_dims,mode", [
    (BF, 128, 32, 8, 64, [(300, 300)], 1e-6, True, 128, Z.ROPE_NEOX),
    (HF, 128, 8, 2, 16, [(1, 40), (1, 16), (1, 1), (1, 17)], 1e-6, True, 128, Z.ROPE_NEOX),
    (BF, 64, 8, 4, 16, [(5, 50), (0, 9), (40, 41)], 1e-5, True, 64, Z.ROPE_NORMAL),
    (HF, 256, 6, 2, 32, [(70, 200)], 1e-6, False, 128, Z.ROPE_NEOX),
    (BF, 80, 5, 5, 128, [(33, 140)], -1.0, False, 20, Z.ROPE_NEOX),
    (HF, 96, 4, 1, 256, [(3, 300), (9, 9)], -1.0, False, 0, Z.ROPE_NEOX),
    (BF, 8, 2, 1, 16, [(20, 20)], 1e-6, True, 6, Z.ROPE_NORMAL),
    (BF, 200, 3, 3, 16, [(17, 50)], 0.0, True, 198, Z.ROPE_NEOX),
])
@pytest.mark.parametrize("heads_first", [False, True])
def test_append_equals_the_definition(dt, d, heads, kv_heads, page, lens, eps, weights, n_dims, mode, heads_first):
    g = torch.Generator("cuda").manual_seed(d)
    held = [-(-kv // page) for _, kv in lens]
    pages = sum(held) + 3
    order = random.Random(d).sample(range(pages), pages)
    rows = [[order.pop() for _ in range(n)] for n in held]
    table = i32([r + [-1] * (max(held) - len(r)) for r in rows])
    starts = [2]
    for n, _ in lens:
        starts.append(starts[-1] + n)
    T = starts[-1] + 5  # two rows before the first sequence, five behind the last
    shape = (2, pages, kv_heads, page, d) if heads_first else (2, pages, page, kv_heads, d)
    k, v = (torch.full(shape, 9.0, dtype=dt, device="cuda") for _ in range(2))
    if heads_first:
        k, v = k.transpose(2, 3), v.transpose(2, 3)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g) * 1.5
    kn, vn, q = rnd(T, kv_heads, d), rnd(T, kv_heads * d + 8), rnd(T, heads, d)
    vn = vn[:, :kv_heads * d]
    kw, qw = ((torch.rand(d, device="cuda", generator=g) + 0.5) if weights else None for _ in range(2))
    rope = rope_table([p % 97 for p in range(T)], n_dims) if n_dims else None
    q_out = torch.full((T, heads, d), 9.0, dtype=dt, device="cuda")
    batch = Z.KvBatch(i32(starts), i32([kv for _, kv in lens]), table, T=T, max_q=max(n for n, _ in lens),
                      max_kv=max(kv for _, kv in lens))
    Z.kv_append(Z.KvCache(k, v), 1, batch, kn, vn, q=q, q_out=q_out, k_norm=kw, q_norm=qw, eps=eps, rope=rope,
                mode=mode)
    neox = mode == Z.ROPE_NEOX
    want_k, want_q = turned(kn, kw, eps, rope, neox), turned(q, qw, eps, rope, neox)
    inside = slice(starts[0], starts[-1])
    assert near(q_out[inside], want_q[inside], dt)
    assert (q_out[:2] == 9).all() and (q_out[starts[-1]:] == 9).all()
    written = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
    for s, (n, kv) in enumerate(lens):
        for i in range(n):
            p, t = kv - n + i, starts[s] + i
            at = rows[s][p // page], p % page
            written[at] = True
            assert near(k[1][at], want_k[t], dt)
            assert torch.equal(v[1][at].reshape(-1), vn[t].to(dt))
    assert (k[0] == 9).all() and (v[0] == 9).all()
    assert (k[1][~written] == 9).all() and (v[1][~written] == 9).all()


def test_append_without_queries_and_bad_places():
    kv_heads, d, page = 2, 64, 16
    k, v = (torch.full((1, 4, page, kv_heads, d), 9.0, dtype=BF, device="cuda") for _ in range(2))
    kn, vn = torch.randn(6, kv_heads, d, device="cuda"), torch.randn(6, kv_heads, d, device="cuda")
    cache, err = Z.KvCache(k, v), torch.zeros(1, dtype=torch.int32, device="cuda")
    # sequences of two rows: one whole, one whose page is none, one of fewer tokens than it has new ones
    batch = Z.KvBatch(i32([0, 2, 4, 6]), i32([18, 2, 1]), i32([[0, 2], [7, -1], [3, -1]]), T=6, max_q=2, max_kv=40)
    Z.kv_append(cache, 0, batch, kn, vn, err=err)
    assert int(err) == Z.ERR_BAD_PAGE | Z.ERR_BAD_SEQ
    assert torch.equal(k[0, 2, :2], kn[:2].to(BF)) and torch.equal(v[0, 2, :2], vn[:2].to(BF))
    assert torch.equal(k[0, 3, 0], kn[5].to(BF))
    assert (k[0, :2] == 9).all() and (k[0, 2, 2:] == 9).all() and (k[0, 3, 1:] == 9).all()


def test_append_rounds_once_at_the_types_ends():
    """Infinities and NaN pass through, f16 overflows to infinity, ties go to even."""
    x = torch.tensor([math.inf, -math.inf, math.nan, 65519.0, 65520.0, 1 + 2.0 ** -9, 1 + 3 * 2.0 ** -9, 2.0 ** -25],
                     device="cuda")
    for dt in (BF, HF):
        k, v = (torch.zeros(1, 1, 16, 1, 8, dtype=dt, device="cuda") for _ in range(2))
        batch = Z.KvBatch(i32([0, 1]), i32([1]), i32([[0]]), T=1, max_q=1, max_kv=1)
        Z.kv_append(Z.KvCache(k, v), 0, batch, x[None, None], x[None, None])
        for got in (k, v):
            assert torch.equal(got[0, 0, 0, 0].nan_to_num(nan=5.0), x.to(dt).nan_to_num(nan=5.0))


class Tables:
    """The same tables on the device and on the host."""

    def __init__(self, pages, seqs, width, page, layers=2, kv_heads=2, d=64, heads_first=False, apart=False):
        self.host = Pages(pages, seqs, width, page)
        g = torch.Generator("cuda").manual_seed(pages)
        shape = (layers, pages, kv_heads, page, d) if heads_first else (layers, pages, page, kv_heads, d)
        if apart:  # heads of d inside rows of d + 8
            shape = shape[:-1] + (d + 8,)
        self.k, self.v = (torch.randn(shape, device="cuda", generator=g).to(BF)[..., :d] for _ in range(2))
        if heads_first:
            self.k, self.v = self.k.transpose(2, 3), self.v.transpose(2, 3)
        self.cache = Z.KvCache(self.k, self.v)
        self.t = Z.KvTables(i32(self.host.refs), i32(self.host.table), i32(self.host.len))

    def agree(self, t=None):
        refs, table, lens = (x.tolist() for x in (t or self.t).tensors)
        assert refs == self.host.refs and table == self.host.table and lens == self.host.len

    def step(self, name, *args, fresh=False):
        """One operation on both sides, in place or into other arrays; the pools too."""
        k, v = self.k.clone(), self.v.clone()
        moves = getattr(self.host, name)(*args)
        for a, b in moves:
            k[:, b], v[:, b] = k[:, a], v[:, a]
        before = [x.clone() for x in self.t.tensors]
        out = Z.KvTables(*(torch.full_like(x, 77) for x in self.t.tensors)) if fresh else None
        got = getattr(Z, "kv_" + name)(self.cache, self.t, *(i32(a) for a in args), out=out)
        self.agree(got)
        if fresh:
            assert all(torch.equal(a, b) for a, b in zip(before, self.t.tensors))
        self.t = got
        assert torch.equal(self.k, k) and torch.equal(self.v, v)
        return moves


@pytest.mark.parametrize("pages,seqs,width,page,kw", [
    (60, 9, 12, 16, {}), (300, 20, 40, 16, dict(heads_first=True, d=80)), (9000, 40, 300, 32, dict(kv_heads=1, d=8)),
    (60, 9, 12, 64, dict(apart=True, kv_heads=3, d=72)), (40, 5, 20, 256, dict(layers=1))])
@pytest.mark.parametrize("fresh", [False, True])
def test_page_operations_follow_the_model(pages, seqs, width, page, kw, fresh):
    t = Tables(pages, seqs, width, page, **kw)
    r = random.Random(pages + fresh)
    moved = 0
    for _ in range(40):
        free = sum(x == 0 for x in t.host.refs)
        empty = [s for s in range(seqs) if t.host.len[s] == 0]
        full = [s for s in range(seqs) if t.host.len[s]]
        op = r.choice(["grow", "grow", "fork", "free", "compact"])
        if op == "grow":
            who = r.sample(range(seqs), r.randint(1, max(1, seqs // 2)))
            room = [width * page - t.host.len[s] for s in who]
            add = [r.randint(0, max(0, min(x, page * (free // len(who) - 1)))) for x in room]
            t.step("grow", who, add, fresh=fresh)
        elif op == "fork" and full and empty:
            dst = r.sample(empty, r.randint(1, min(3, len(empty))))
            if free >= len(dst):
                moved += len(t.step("fork", [r.choice(full) for _ in dst], dst, fresh=fresh))
        elif op == "free" and full:
            who = r.sample(full, r.randint(1, len(full)))
            t.step("free", who, fresh=fresh)
        elif op == "compact":
            moved += len(t.step("compact", fresh=fresh))
    assert moved > 0


def test_large_tables_out_of_place():
    """Tables beyond what one block copies, and a pool of several scan steps."""
    t = Tables(20000, 300, 400, 16, layers=1, kv_heads=1, d=8)
    r = random.Random(1)
    t.step("grow", list(range(0, 300, 2)), [r.randint(1, 1500) for _ in range(150)], fresh=True)
    t.step("fork", [0] * 60 + [2] * 60, list(range(1, 240, 2)), fresh=True)
    t.step("free", list(range(0, 150)), fresh=True)
    t.step("compact", fresh=True)


@pytest.mark.parametrize("fresh", [False, True])
def test_the_most_sequences_of_a_call(fresh):
    """1,024 at once, each of which takes pages, is copied with a part page, and is freed."""
    n = Z.KV_MAX_SEQS
    t = Tables(5 * n, 2 * n + 3, 4, 16, layers=1, kv_heads=1, d=8)
    r = random.Random(7)
    order = r.sample(range(2 * n), 2 * n)
    t.step("grow", order[:n], [r.randint(1, 40) for _ in range(n)], fresh=fresh)
    assert len(t.step("fork", order[:n], order[n:], fresh=fresh)) > n // 2
    t.step("free", order[:n], fresh=fresh)
    assert t.step("compact", fresh=fresh)
    with pytest.raises(Z.ZestError, match="0 to 1024"):
        Z.kv_free(t.cache, t.t, i32(list(range(n + 1))))


@pytest.mark.parametrize("fresh", [False, True])
def test_tables_that_start_anywhere(fresh):
    """Arrays 4 bytes past a 16-byte boundary, and of lengths that are no multiple of four."""
    def shifted(x):
        at = torch.full((x.numel() + 1,), 55, dtype=torch.int32, device="cuda")
        at[1:] = x.flatten()
        return at[1:].view(x.shape)

    t = Tables(131, 11, 13, 16)
    t.t = Z.KvTables(*(shifted(x) for x in t.t.tensors))
    t.step("grow", [0, 3, 7], [100, 200, 33], fresh=fresh)
    t.step("fork", [3, 7, 3], [1, 2, 4], fresh=fresh)
    t.step("free", [0, 3], fresh=fresh)
    t.step("compact", fresh=fresh)
    assert fresh or all(int(x.flatten().as_strided((1,), (1,), 0)) == 55 for x in t.t.tensors)


@pytest.mark.parametrize("fresh", [False, True])
def test_page_operations_that_fail_change_nothing(fresh):
    t = Tables(10, 6, 8, 16)
    t.step("grow", [0, 1], [100, 20])  # 7 + 2 pages of 10
    fails = [("grow", ([2, 3], [16, 17]), Z.ERR_NO_PAGES), ("grow", ([0], [30]), Z.ERR_BAD_SEQ),
             ("grow", ([2, 2], [1, 1]), Z.ERR_BAD_SEQ), ("grow", ([6], [1]), Z.ERR_BAD_SEQ),
             ("grow", ([-1], [1]), Z.ERR_BAD_SEQ), ("grow", ([0], [-1]), Z.ERR_BAD_SEQ),
             ("grow", ([2], [0x7fffffff]), Z.ERR_BAD_SEQ),
             ("fork", ([0, 1], [2, 3]), Z.ERR_NO_PAGES), ("fork", ([0], [1]), Z.ERR_BAD_SEQ),
             ("fork", ([0, 1], [2, 2]), Z.ERR_BAD_SEQ), ("fork", ([9], [2]), Z.ERR_BAD_SEQ),
             ("fork", ([0], [-2]), Z.ERR_BAD_SEQ), ("free", ([0, 6],), Z.ERR_BAD_SEQ),
             ("free", ([-1],), Z.ERR_BAD_SEQ)]
    k, v = t.k.clone(), t.v.clone()
    for name, args, bit in fails:
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        out = Z.KvTables(*(torch.full_like(x, 77) for x in t.t.tensors)) if fresh else None
        got = getattr(Z, "kv_" + name)(t.cache, t.t, *(i32(a) for a in args), out=out, err=err)
        assert int(err) == bit, name
        t.agree(got)
    assert torch.equal(t.k, k) and torch.equal(t.v, v)
    with pytest.raises(Z.ZestError, match="error bits 0x10"):
        Z.kv_grow(t.cache, t.t, i32([2]), i32([60]))
    # a page number that is none, in a row to be copied or given back
    t.t.tensors[1][1, 0] = 10
    before = [x.clone() for x in t.t.tensors]
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    Z.kv_fork(t.cache, t.t, i32([1]), i32([4]), err=err)
    assert int(err) == Z.ERR_BAD_PAGE and all(torch.equal(a, b) for a, b in zip(before, t.t.tensors))
    Z.kv_free(t.cache, t.t, i32([1]), err=err)
    assert int(err) == Z.ERR_BAD_PAGE and t.t.tensors[2].tolist()[1] == 0


@pytest.mark.parametrize("pages,seqs,width", [(40, 6, 9), (40, 7000, 10)])
@pytest.mark.parametrize("fresh", [False, True])
def test_a_compaction_that_fails_changes_nothing(pages, seqs, width, fresh):
    """A table with an entry that is no page, small and large enough to be looked over apart: tables and pools stay,
    and the same call without the entry goes through."""
    t = Tables(pages, seqs, width, 16)
    t.step("grow", [0, 1, 5], [100, 130, 60])
    t.step("free", [0])
    good = t.t.tensors[1].clone()
    for at, entry in (((3, 2), pages), ((seqs - 1, width - 1), 0x7fffffff), ((0, 0), pages + 1)):
        t.t.tensors[1][at] = entry
        before, k, v = [x.clone() for x in t.t.tensors], t.k.clone(), t.v.clone()
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        out = Z.KvTables(*(torch.full_like(x, 77) for x in t.t.tensors)) if fresh else None
        got = Z.kv_compact(t.cache, t.t, out=out, err=err)
        assert int(err) == Z.ERR_BAD_PAGE
        assert all(torch.equal(a, b) for a, b in zip(before, got.tensors))
        assert all(torch.equal(a, b) for a, b in zip(before, t.t.tensors))
        assert torch.equal(t.k, k) and torch.equal(t.v, v)
        t.t.tensors[1].copy_(good)
    assert t.step("compact", fresh=fresh)


@pytest.mark.parametrize("fresh", [False, True])
def test_a_row_gone_bad_is_freed(fresh):
    """Entries that are no page, and a page nobody holds: dropped with an error bit; the rest of the row, and the
    other sequences named, are given back."""
    t = Tables(30, 6, 9, 16)
    t.step("grow", [0, 1, 2], [100, 70, 40])
    t.step("fork", [0], [4])
    refs, table, lens = t.t.tensors
    table[1, 1], table[1, 6], table[0, 8] = 30, 0x7fffffff, 29  # page 29 is free
    held = t.host.table[1][1]
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = Z.KvTables(*(torch.full_like(x, 77) for x in t.t.tensors)) if fresh else None
    got = Z.kv_free(t.cache, t.t, i32([1, 0]), out=out, err=err)
    assert int(err) == Z.ERR_BAD_PAGE
    t.host.free([0, 1])
    t.host.refs[held] += 1  # its row no longer said so
    t.agree(got)


def test_the_same_sequence_twice():
    t = Tables(30, 8, 8, 16)
    t.step("grow", [0, 1], [40, 33])
    t.step("fork", [0, 0, 1], [2, 3, 4])
    t.step("free", [0, 2])
    host = t.host
    host.free([3, 1])
    Z.kv_free(t.cache, t.t, i32([3, 1, 3, 3, 1]))
    t.agree()
    # no sequence at all, and an empty one
    t.step("free", [])
    t.step("fork", [5], [6])
    t.step("grow", [], [])


def test_captured_page_operations():
    """Each of them in one graph, replayed over other sequences and counts."""
    t = Tables(80, 8, 12, 16)
    t.step("grow", [0, 1, 2], [60, 77, 33])
    arrays = {name: torch.zeros(2, dtype=torch.int32, device="cuda") for name in ("seq", "add", "src", "dst", "gone")}
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    ws = torch.empty(Z.lib().zest_kv_pages_workspace(t.cache.ref), dtype=torch.uint8, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        Z.kv_grow(t.cache, t.t, arrays["seq"], arrays["add"], err=err)
        Z.kv_fork(t.cache, t.t, arrays["src"], arrays["dst"], workspace=ws, err=err)
        Z.kv_free(t.cache, t.t, arrays["gone"], err=err)
        Z.kv_compact(t.cache, t.t, workspace=ws, err=err)
    t.agree()  # nothing has run
    for seq, add, src, dst, gone in [([0, 2], [5, 20], [0, 1], [3, 4], [0, 1]), ([3, 4], [40, 1], [2, 3], [0, 1], [2, 4]),
                                     ([0, 1], [1, 1], [1, 1], [5, 6], [3, 1])]:
        for name, v in dict(seq=seq, add=add, src=src, dst=dst, gone=gone).items():
            arrays[name].copy_(i32(v))
        k, v = t.k.clone(), t.v.clone()
        for moves in (t.host.grow(seq, add), t.host.fork(src, dst), t.host.free(gone), t.host.compact()):
            for a, b in moves:
                k[:, b], v[:, b] = k[:, a], v[:, a]
        g.replay()
        t.agree()
        assert int(err) == 0 and torch.equal(t.k, k) and torch.equal(t.v, v)


def test_offsets_past_32_bits():
    """Pools of two layers whose last pages lie past 2^32 values: written, copied and moved there, and nowhere else."""
    layers, page, kv_heads, d = 2, 64, 8, 128
    pages = (1 << 31) // (page * kv_heads * d) + 40
    k, v = (torch.zeros(layers, pages, page, kv_heads, d, dtype=BF, device="cuda") for _ in range(2))
    cache, last = Z.KvCache(k, v), pages - 1
    assert (k[1, last - 2].data_ptr() - k.data_ptr()) // 2 > 1 << 32
    g = torch.Generator("cuda").manual_seed(2)
    kn, vn = (torch.randn(100, kv_heads, d, device="cuda", generator=g) for _ in range(2))
    batch = Z.KvBatch(i32([0, 100]), i32([100]), i32([[last, last - 2]]), T=100, max_q=100, max_kv=100)
    for layer in range(layers):
        Z.kv_append(cache, layer, batch, kn, vn)
        for x, new in ((k, kn), (v, vn)):
            assert torch.equal(x[layer, last], new[:64].to(BF)) and torch.equal(x[layer, last - 2, :36], new[64:].to(BF))
    used = lambda x: x.view(layers, pages, -1).view(torch.int64).ne(0).any(-1)
    where = torch.zeros(layers, pages, dtype=torch.bool)
    where[:, [last, last - 2]] = True
    assert torch.equal(used(k).cpu(), where) and torch.equal(used(v).cpu(), where)
    # a fork whose one free page is the last but one: the part page is copied to it
    refs = torch.ones(pages, dtype=torch.int32, device="cuda")
    refs[last - 1] = 0
    t = Z.KvTables(refs, i32([[last, last - 2], [-1, -1]]), i32([100, 0]))
    Z.kv_fork(cache, t, i32([0]), i32([1]))
    assert t.tensors[1].tolist() == [[last, last - 2], [last, last - 1]] and t.tensors[2].tolist() == [100, 100]
    assert torch.equal(k[:, last - 1], k[:, last - 2]) and torch.equal(v[:, last - 1], v[:, last - 2])
    # only these three in use: they move to the front
    refs.zero_()
    refs[last - 2], refs[last - 1], refs[last] = 1, 1, 2
    kept = k[:, last - 2:].clone(), v[:, last - 2:].clone()
    Z.kv_compact(cache, t)
    assert t.tensors[1].tolist() == [[2, 0], [2, 1]] and refs[:4].tolist() == [1, 1, 2, 0] and int(refs.sum()) == 4
    assert torch.equal(k[:, :3], kept[0]) and torch.equal(v[:, :3], kept[1])
    where[:, :3] = True
    where[:, last - 1] = True
    assert torch.equal(used(k).cpu(), where) and torch.equal(used(v).cpu(), where)


def test_a_serving_loop():
    """Prompts in chunks, forks, single tokens, ended sequences, compaction: every step's attention against the
    attention of what the sequences hold, with the operators run together, the tables never read by the host."""
    layers, page, heads, kv_heads, d, seqs, width, pages = 2, 16, 8, 2, 64, 6, 24, 90
    t = Tables(pages, seqs, width, page, layers=layers, kv_heads=kv_heads, d=d)
    r, g = random.Random(4), torch.Generator("cuda").manual_seed(4)
    held = {s: [torch.zeros(2, 0, kv_heads, d, dtype=BF, device="cuda") for _ in range(layers)] for s in range(seqs)}
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    ws = torch.empty(32 << 20, dtype=torch.uint8, device="cuda")
    w = torch.rand(d, device="cuda", generator=g) + 0.5

    def step(who, new):
        """Sequences `who` get new tokens each: grown, appended and attended in every layer."""
        Z.kv_grow(t.cache, t.t, i32(who), i32(new), err=err)
        t.host.grow(who, new)
        T = sum(new)
        starts = [sum(new[:i]) for i in range(len(new) + 1)]
        index = torch.tensor(who, device="cuda")
        batch = Z.KvBatch(i32(starts), t.t.tensors[2][index].contiguous(), t.t.tensors[1][index].contiguous(), T=T,
                          max_q=max(new), max_kv=width * page)
        pos = [t.host.len[s] - n + i for s, n in zip(who, new) for i in range(n)]
        rope = rope_table(pos, d)
        for layer in range(layers):
            rnd = lambda h: torch.randn(T, h, d, device="cuda", generator=g)
            q, k, v = rnd(heads), rnd(kv_heads), rnd(kv_heads)
            q16 = torch.empty(T, heads, d, dtype=BF, device="cuda")
            Z.kv_append(t.cache, layer, batch, k, v, q=q, q_out=q16, k_norm=w, q_norm=w, eps=1e-6, rope=rope, err=err)
            got = Z.kv_attend(t.cache, layer, batch, q16, err=err, workspace=ws)
            assert near(q16, turned(q, w, 1e-6, rope, True), BF)
            for i, s in enumerate(who):
                a, b = starts[i], starts[i + 1]
                # keys as the cache holds them: the last new ones, checked by append's own test
                row, n = t.host.table[s], t.host.len[s]
                at = torch.tensor([row[p // page] * page + p % page for p in range(n)], device="cuda")
                kc, vc = (x[layer].reshape(-1, kv_heads, d)[at] for x in (t.k, t.v))
                old = held[s][layer]
                assert torch.equal(kc[:old.shape[1]], old[0]) and torch.equal(vc[:old.shape[1]], old[1])
                assert torch.equal(vc[old.shape[1]:], v[a:b].to(BF))
                assert near(kc[old.shape[1]:], turned(k[a:b], w, 1e-6, rope[a:b], True), BF)
                held[s][layer] = torch.stack([kc, vc])
                want, mean, _ = attention(q16[a:b].double(), kc.double(), vc.double(), n - (b - a), d ** -0.5, True, 0)
                tol = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -11) * mean
                assert bool(((got[a:b].double() - want).abs() <= tol).all())

    step([0, 1], [70, 45])       # prompts
    step([0], [60])              # a second chunk
    t.step("fork", [0, 0, 1], [2, 3, 4])
    for a, b in ((0, 2), (0, 3), (1, 4)):
        held[b] = [x.clone() for x in held[a]]
    for _ in range(20):          # one token each, some ended and compacted on the way
        step([s for s in range(5) if t.host.len[s]], [1] * sum(t.host.len[s] > 0 for s in range(5)))
        if _ == 8:
            t.step("free", [0, 3])
            for s in (0, 3):
                held[s] = [torch.zeros(2, 0, kv_heads, d, dtype=BF, device="cuda") for _ in range(layers)]
            assert t.step("compact")
    step([5, 2, 3], [33, 1, 7])  # a new prompt beside an old sequence's token
    assert int(err) == 0
    t.agree()
