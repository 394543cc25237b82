"""zest_kv_attend against the attention's definition in 64 bits: types, head
layouts, lengths, page sizes, masks, strides, values that must not reach a
row, captured and concurrent calls.

Tolerance, per value: the output's own rounding, half a step of the value
(eps / 2 * |o|); the weights' rounding to the cache's type before they meet
the values, half a step of each (eps / 2 * sum p |v| / sum p); and f32: the
scores are d-term f32 sums of products of magnitude |q||k| scale, at most
d 2^-24 of the largest such sum here (|score| below 2^5: 256 * 2^-24 * 2^5 =
2^-11 in the worst case and about its square root's share, 2^-15, in fact),
the exponential and the running sums a few 2^-22: together below 2^-11 of
sum p |v| / sum p. f16 weights below 2^-14 are held to 2^-25 absolutely,
relative to a largest weight of 2^-8 to 1."""
import math
import random
import subprocess
import sys

import pytest
import torch

import zest_b200 as Z
from kv_util import attention, laid_out

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Case:
    """A batch of (new tokens, all tokens) over a pool whose pages lie in no order, NaN in everything that no
    sequence holds."""

    def __init__(self, lens, heads, kv_heads, d, page, dt, seed=0, heads_first=False, spare=2, width=None, layers=1):
        g = torch.Generator("cuda").manual_seed(seed)
        self.lens, self.heads, self.kv_heads, self.d, self.page, self.dt = lens, heads, kv_heads, d, page, dt
        held = [-(-kv // page) for _, kv in lens]
        pages = sum(held) + spare
        order = random.Random(seed).sample(range(pages), pages)
        self.width = width or max([1] + held)
        self.rows = []
        for n in held:
            self.rows.append([order.pop() for _ in range(n)])
        self.table = i32([r + [-1] * (self.width - len(r)) for r in self.rows])
        starts = [0]
        for n, _ in lens:
            starts.append(starts[-1] + n)
        self.T = starts[-1]
        self.starts = starts
        self.q_start, self.kv_len = i32(starts), i32([kv for _, kv in lens])
        shape = (layers, pages, kv_heads, page, d) if heads_first else (layers, pages, page, kv_heads, d)
        pool = lambda: (torch.randn(shape, device="cuda", generator=g) * 1.1).to(dt)
        self.k, self.v = pool(), pool()
        if heads_first:
            self.k, self.v = self.k.transpose(2, 3), self.v.transpose(2, 3)
        mine = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
        for row, (_, kv) in zip(self.rows, lens):
            for j, p in enumerate(row):
                mine[p, :min(page, kv - j * page)] = True
        self.k[:, ~mine] = math.nan
        self.v[:, ~mine] = math.nan
        self.q = torch.randn(self.T, heads, d, device="cuda", generator=g).to(dt)
        self.max_q, self.max_kv = max([n for n, _ in lens] + [0]), max([kv for _, kv in lens] + [0])
        self.cache = Z.KvCache(self.k, self.v)
        self.batch = Z.KvBatch(self.q_start, self.kv_len, self.table, T=self.T, max_q=self.max_q, max_kv=self.max_kv)
        self.scale = 1 / math.sqrt(d)

    def want(self, causal=True, window=0, layer=0):
        o = torch.zeros(self.T, self.heads, self.d, dtype=torch.float64, device="cuda")
        a, n = torch.zeros_like(o), torch.zeros(self.T, dtype=torch.int64, device="cuda")
        for s, (new, kv) in enumerate(self.lens):
            i, j = self.starts[s], self.starts[s + 1]
            k, v = (laid_out(x[layer], self.rows[s], kv, self.page) for x in (self.k, self.v))
            o[i:j], a[i:j], n[i:j] = attention(self.q[i:j].double(), k, v, kv - new, self.scale, causal, window)
        return o, a, n

    def check(self, got, causal=True, window=0, layer=0, eps=None):
        o, a, n = self.want(causal, window, layer)
        e = torch.finfo(self.dt).eps / 2
        out = e if eps is None else eps
        tol = out * o.abs() + (e + 2 ** -11) * a + 1e-30
        if self.dt == HF:
            tol += n[:, None, None] * 2.0 ** -25 * 2 ** 8 * 4 / n.clamp(min=1)[:, None, None].double().sqrt() + 2 ** -25
        got = got.double().view(o.shape)
        assert torch.equal(torch.isfinite(got), torch.isfinite(o)), "another set of finite values"
        fine = torch.isfinite(o)
        worst = ((got - o).abs() / tol)[fine]
        assert worst.numel() == 0 or worst.max().item() <= 1.0, f"{worst.max().item():.3g} times the tolerance"


FEW = [  # up to 16 rows of a kv head, and a few tiles of them
    (BF, 128, 32, 8, 64, [(1, 1000)], True, 0),
    (HF, 128, 32, 8, 16, [(1, 1), (1, 17), (1, 64), (1, 65), (1, 700)], True, 0),
    (BF, 64, 32, 8, 16, [(1, 5), (2, 300), (4, 4), (3, 90)], True, 0),
    (HF, 256, 24, 4, 64, [(1, 900), (2, 33)], True, 0),
    (BF, 128, 8, 8, 32, [(1, 50), (5, 200)], True, 0),          # one query head a kv head
    (BF, 128, 12, 2, 128, [(1, 513), (2, 1)], True, 0),         # fewer keys than new tokens
    (HF, 96, 15, 3, 256, [(3, 300), (1, 256)], True, 0),
    (BF, 8, 2, 1, 16, [(1, 40), (7, 40)], True, 0),
    (HF, 72, 9, 9, 16, [(1, 129)], False, 0),
    (BF, 128, 16, 1, 64, [(1, 400)], True, 100),
    (BF, 80, 6, 2, 16, [(1, 200), (3, 77), (1, 3)], True, 1),
    (HF, 128, 8, 2, 64, [(1, 4000)], True, 37),
]
MANY = [  # chunks of new tokens
    (BF, 128, 8, 2, 64, [(300, 300)], True, 0),
    (BF, 128, 8, 2, 64, [(257, 1000)], True, 0),
    (HF, 128, 4, 4, 16, [(130, 513)], True, 0),
    (HF, 64, 8, 2, 16, [(100, 400), (1, 90), (0, 50), (33, 33)], True, 0),
    (BF, 64, 12, 2, 32, [(200, 260)], True, 50),
    (BF, 256, 6, 1, 64, [(90, 333)], True, 0),
    (HF, 256, 4, 2, 128, [(140, 140), (70, 200)], True, 0),
    (BF, 128, 14, 2, 256, [(64, 600)], True, 0),                # 7 query heads a kv head
    (HF, 112, 10, 2, 64, [(65, 129)], True, 0),
    (BF, 128, 71, 1, 64, [(20, 200)], True, 0),                 # one kv head for 71
    (BF, 128, 8, 2, 64, [(150, 40)], True, 0),                  # rows before the first key: zeros
    (BF, 128, 8, 2, 64, [(150, 0), (40, 0)], True, 0),
    (HF, 128, 8, 2, 64, [(100, 333), (40, 1)], False, 0),       # to an encoder's states
    (BF, 200, 4, 2, 16, [(70, 300)], False, 0),
    (BF, 128, 8, 8, 16, [(300, 2000)], True, 200),
    (HF, 64, 4, 1, 64, [(513, 700)], True, 3),
]


@pytest.mark.parametrize("dt,d,heads,kv_heads,page,lens,causal,window", FEW + MANY)
def test_equals_the_definition(dt, d, heads, kv_heads, page, lens, causal, window):
    c = Case(lens, heads, kv_heads, d, page, dt, seed=d + heads)
    c.check(Z.kv_attend(c.cache, 0, c.batch, c.q, causal=causal, window=window), causal, window)


@pytest.mark.parametrize("dt,d,heads,kv_heads,page,lens,causal,window", [
    (BF, 256, 6, 1, 128, [(39, 3068), (39, 3068)], True, 0), (HF, 256, 24, 4, 64, [(500, 3000)], True, 0),
    (BF, 256, 8, 8, 16, [(190, 4000), (19, 2000)], False, 0), (BF, 200, 32, 8, 32, [(300, 2500)], True, 400),
    (HF, 128, 16, 4, 16, [(600, 4000), (33, 1000)], True, 0), (BF, 64, 16, 4, 16, [(600, 4000), (33, 1000)], True, 0)])
def test_many_tiles_one_after_another(dt, d, heads, kv_heads, page, lens, causal, window):
    """Long enough for every buffer to be used many times over, several times."""
    c = Case(lens, heads, kv_heads, d, page, dt, seed=d)
    for _ in range(4):
        c.check(Z.kv_attend(c.cache, 0, c.batch, c.q, causal=causal, window=window), causal, window)


@pytest.mark.parametrize("lens", [[(1, 3000)], [(1, 5000), (1, 100), (1, 2500)], [(40, 3000)], [(200, 6000)]])
@pytest.mark.parametrize("heads_first", [False, True])
def test_long_keys_are_cut_and_joined(lens, heads_first):
    c = Case(lens, 8, 2, 128, 16, BF, seed=5, heads_first=heads_first)
    c.check(Z.kv_attend(c.cache, 0, c.batch, c.q))
    # the launch is shaped by the bounds, the result is not
    wide = Z.KvBatch(c.q_start, c.kv_len, c.table, T=c.T, max_q=c.max_q + 100, max_kv=c.max_kv * 9)
    c.check(Z.kv_attend(c.cache, 0, wide, c.q))


@pytest.mark.parametrize("dt,d,kv_heads,page,lens,causal,window", [
    (BF, 128, 2, 64, [(1, 8192)], True, 0), (HF, 128, 2, 16, [(1, 8192), (1, 8192), (1, 700)], True, 0),
    (BF, 64, 4, 32, [(2, 8192)], True, 0), (HF, 256, 1, 128, [(1, 8000), (1, 90)], True, 0),
    (BF, 128, 2, 64, [(40, 8192)], False, 0), (HF, 64, 4, 16, [(70, 8192)], True, 0),
    (BF, 256, 2, 64, [(30, 16000)], True, 0), (HF, 128, 2, 64, [(200, 8000), (33, 5000)], True, 0),
    (BF, 128, 2, 64, [(2100, 8192)], True, 0), (BF, 128, 2, 16, [(1, 8100)], True, 5000),
    (HF, 128, 2, 16, [(60, 8100)], True, 5001)])
def test_no_key_is_lost_or_doubled_at_a_cut(dt, d, kv_heads, page, lens, causal, window):
    """Queries of zero weigh every key a row sees alike: with one value of 4096 in a column and zeros in the rest, the
    column is 4096 / (the keys it sees), or zero where that key is not seen. A column each for the keys on both sides
    of every multiple of 64, where keys may be cut into parts, rings and tiles end. The weights are 1 to 2^-20 and
    round to 1, the sum of them is within 2^-18, the result is rounded once: eps / 2 + 2^-16 of the value."""
    c = Case(lens, 4 * kv_heads, kv_heads, d, page, dt, seed=31)
    c.q.zero_()
    c.v[0][torch.isfinite(c.v[0])] = 0.0
    want = torch.zeros(c.T, kv_heads, d, dtype=torch.float64, device="cuda")
    for s, (n, kv) in enumerate(lens):
        pos = torch.arange(kv - n, kv, device="cuda") if causal else torch.full((n,), kv - 1, device="cuda")
        low = (pos - window + 1).clamp(min=0) if window else torch.zeros_like(pos)
        keys = [x for m in range(0, kv + 64, 64) for x in (m - 1, m) if 0 <= x < kv]
        first = max(0, len(keys) - kv_heads * d)  # more than there are columns: the last of them
        for i, key in enumerate(keys[first:]):
            head, col = i // d, i % d
            c.v[0, c.rows[s][key // page], key % page, head, col] = 4096.0
            sees = (key <= pos) & (key >= low)
            want[c.starts[s]:c.starts[s + 1], head, col] = torch.where(sees, 4096.0 / (pos - low + 1), 0.0)
    want = want.repeat_interleave(4, 1)
    got = Z.kv_attend(c.cache, 0, c.batch, c.q, causal=causal, window=window).double()
    assert bool(((got - want).abs() <= (torch.finfo(dt).eps / 2 + 2.0 ** -16) * want).all())


@pytest.mark.parametrize("lens", [[(1, 200)], [(1, 3000)], [(150, 400)]])
def test_outputs_and_strides(lens):
    c = Case(lens, 8, 2, 128, 64, BF, seed=9, layers=3)
    W = 8 * 128
    q = torch.full((c.T, W + 24), math.nan, dtype=BF, device="cuda")
    q[:, :W] = c.q.view(c.T, W)
    out = torch.full((c.T, W + 40), 7.0, dtype=BF, device="cuda")
    y = torch.full((c.T, W + 4), 7.0, device="cuda")
    a = torch.full((c.T, W + 8), 7, dtype=torch.int16, device="cuda")
    Z.kv_attend(c.cache, 2, c.batch, q[:, :W], out=out[:, :W], y=y[:, :W], a_next=a[:, :W])
    c.check(y[:, :W], layer=2, eps=2.0 ** -23)
    assert torch.equal(out[:, :W], y[:, :W].to(BF))
    _, want = Z.pack_activations(y[:, :W].contiguous(), want_bytes=False)
    assert torch.equal(a[:, :W], want[:c.T])
    assert (out[:, W:] == 7).all() and (y[:, W:] == 7).all() and (a[:, W:] == 7).all()
    again = torch.empty((c.T, W), device="cuda")
    Z.kv_attend(c.cache, 2, c.batch, q[:, :W], y=again)
    assert torch.equal(again, y[:, :W])


@pytest.mark.parametrize("d,lens,window", [(128, [(5, 100)], 0), (128, [(200, 300)], 0), (64, [(90, 300)], 20),
                                           (256, [(70, 200)], 0), (128, [(3, 3000)], 0), (256, [(2, 130)], 40)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_values_a_row_does_not_see_do_not_reach_it(d, lens, window, bad):
    c = Case(lens, 8, 2, d, 16, BF, seed=3)
    n, kv = lens[0]
    at = lambda p: (c.rows[0][p // 16], p % 16)
    # in the last token's value, one before it, and (seen by the first rows alone) at the window's start
    for p, head, col in [(kv - 1, 0, 3), (kv - 2, 1, d - 1)] + ([(kv - n - window + 1, 0, 5)] if window else []):
        c.v[0][at(p)][head, col] = bad
    c.check(Z.kv_attend(c.cache, 0, c.batch, c.q, window=window), window=window)
    # a NaN or infinite key reaches the rows that see it alone
    c = Case(lens, 8, 2, d, 16, BF, seed=4)
    c.k[0][at(kv - 1)][1, 2] = math.nan
    got = Z.kv_attend(c.cache, 0, c.batch, c.q, window=window)
    assert torch.isnan(got[n - 1, 4:]).all()
    rest = torch.ones(n, 8, dtype=torch.bool, device="cuda")
    rest[n - 1, 4:] = False
    assert torch.isfinite(got[rest]).all()


@pytest.mark.parametrize("d,lens,window", [(128, [(64, 64)], 0), (64, [(64, 640)], 0), (96, [(61, 200), (64, 70)], 30),
                                           (128, [(64, 6000)], 0)])
def test_not_finite_values_in_the_last_tile_of_two_query_tiles(d, lens, window):
    """A block's two query tiles of 32 tokens over one tile of values with NaN and infinities that the first rows of
    either, or all of one, do not see: every row gets what it sees, call after call."""
    c = Case(lens, 8, 2, d, 16, BF, seed=17)
    for s, (n, kv) in enumerate(lens):
        for x, back in enumerate((1, 2, 17, 30, 33, 48, 60)):
            p = kv - back
            c.v[0, c.rows[s][p // 16], p % 16, x % 2, 5 * x] = (math.nan, math.inf, -math.inf)[x % 3]
    first = Z.kv_attend(c.cache, 0, c.batch, c.q, window=window)
    c.check(first, True, window)
    for _ in range(50):
        assert torch.equal(Z.kv_attend(c.cache, 0, c.batch, c.q, window=window).view(torch.int16),
                           first.view(torch.int16))


@pytest.mark.parametrize("d", [64, 128, 96, 256])
@pytest.mark.parametrize("n,window", [(1, 50), (3, 77), (40, 30), (150, 100)])
def test_pages_behind_the_window_may_be_gone(n, window, d):
    """Pages that no row of the step sees any more: their entries none, or out of the pool."""
    c = Case([(n, 700), (n, 333)], 8, 2, d, 16, BF, seed=21)
    want = c.want(True, window)
    for s, (new, kv) in enumerate(c.lens):
        gone = max(0, kv - new - window + 1) // 16
        c.table[s, :gone] = torch.tensor([-1, 1 << 30], dtype=torch.int32, device="cuda").repeat(gone)[:gone]
    c.want = lambda *a: want
    c.check(Z.kv_attend(c.cache, 0, c.batch, c.q, window=window), True, window)
    c.check(Z.kv_attend(c.cache, 0, c.batch, c.q, window=window, workspace=torch.empty(1 << 24, dtype=torch.uint8,
                                                                                    device="cuda")), True, window)


def test_bounds_as_wide_as_they_go():
    """max_q and max_kv of 2^31 - 1 - 4096 cost nothing: no sequence has more than the step's rows or its table row."""
    for lens in ([(1, 900), (2, 40)], [(50, 300)]):
        c = Case(lens, 8, 2, 128, 16, BF, seed=22)
        wide = 0x7fffffff - 4096
        b = Z.KvBatch(c.q_start, c.kv_len, c.table, T=c.T, max_q=wide, max_kv=wide)
        c.check(Z.kv_attend(c.cache, 0, b, c.q))
        c.check(Z.kv_attend(c.cache, 0, b, c.q, window=(1 << 62)))


@pytest.mark.parametrize("lens", [[(6, 3), (2, 60)], [(90, 20), (30, 200)]])
def test_the_widest_window(lens):
    """2^63 - 1, over rows before the first key too: the causal mask alone."""
    c = Case(lens, 8, 2, 128, 16, BF, seed=25)
    c.check(Z.kv_attend(c.cache, 0, c.batch, c.q, window=(1 << 63) - 1))


def test_a_step_of_no_rows():
    """Empty tensors through the binding; and a bound of no rows that a sequence passes."""
    c = Case([(0, 200), (0, 0), (0, 70)], 8, 2, 128, 16, BF, seed=23)
    assert c.q.shape == (0, 8, 128) and Z.kv_attend(c.cache, 0, c.batch, c.q).shape == c.q.shape
    y = torch.empty(0, 8 * 128, device="cuda")
    assert Z.kv_attend(c.cache, 0, c.batch, c.q, y=y) is y
    rows = torch.empty(0, 2, 128, device="cuda")
    Z.kv_append(c.cache, 0, c.batch, rows, rows)
    for lens in ([(1, 200)], [(0, 3000), (1, 3000)]):
        c = Case(lens, 8, 2, 128, 16, BF, seed=24)
        out, err = torch.full_like(c.q, 5.0), torch.zeros(1, dtype=torch.int32, device="cuda")
        b = Z.KvBatch(c.q_start, c.kv_len, c.table, T=c.T, max_q=0, max_kv=c.max_kv)
        Z.kv_attend(c.cache, 0, b, c.q, out=out, err=err)
        assert int(err) == Z.ERR_BAD_SEQ and (out == 5).all()


def test_a_first_call_that_is_captured():
    """A process whose first calls are captured: nothing is set up that a capture forbids."""
    code = """
import sys, torch
sys.path[:0] = ["ggml-xdna_b200", "tests"]
import zest_b200 as Z
from test_gpu_kv_attend import BF, Case
for lens in ([(1, 200)], [(1, 4000)], [(100, 300)]):
    c = Case(lens, 8, 2, 128, 16, BF, seed=1)
    out, err = torch.zeros_like(c.q), torch.zeros(1, dtype=torch.int32, device="cuda")
    ws = torch.empty(1 << 24, dtype=torch.uint8, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        Z.kv_attend(c.cache, 0, c.batch, c.q, out=out, err=err, workspace=ws)
    g.replay()
    torch.cuda.synchronize()
    assert int(err) == 0
    c.check(out)
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=Z.PKG_DIR.parent, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-2000:]


def test_masked_lowest_and_infinite_scores():
    c = Case([(40, 200)], 4, 4, 64, 16, HF, seed=8)
    c.q[:, 0] = 65504.0  # the type's largest: scores of millions, one key takes all
    c.q[:, 1] = 0.0      # every key the same
    c.check(Z.kv_attend(c.cache, 0, c.batch, c.q))


@pytest.mark.parametrize("lens", [[(1, 90), (3, 40)], [(60, 90), (33, 40)]])
def test_rows_outside_the_sequences_stay(lens):
    c = Case(lens, 8, 2, 128, 16, BF, seed=2)
    T = c.T + 150
    q = torch.full((T, 8, 128), math.nan, dtype=BF, device="cuda")
    q[3:3 + c.T] = c.q
    out = torch.full((T, 8, 128), 5.0, dtype=BF, device="cuda")
    b = Z.KvBatch(c.q_start + 3, c.kv_len, c.table, T=T, max_q=c.max_q, max_kv=c.max_kv)
    Z.kv_attend(c.cache, 0, b, q, out=out)
    c.check(out[3:3 + c.T])
    assert (out[:3] == 5).all() and (out[3 + c.T:] == 5).all()


@pytest.mark.parametrize("lens", [[(1, 200), (1, 300), (1, 100)], [(40, 200), (50, 300), (60, 100)]])
def test_bad_sequences_and_pages_raise_bits(lens):
    c = Case(lens, 8, 2, 128, 16, BF, seed=6)
    # under the same bounds: they shape the launch, and with it the order of the sums
    good = Z.kv_attend(c.cache, 0, Z.KvBatch(c.q_start, c.kv_len, c.table, T=c.T, max_q=c.max_q, max_kv=1 << 20), c.q)
    mid = slice(c.starts[1], c.starts[2])
    for change in ("long", "pages", "starts"):
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        out = torch.full_like(good, 5.0)
        kv, table, starts = c.kv_len.clone(), c.table.clone(), c.q_start.clone()
        if change == "long":  # longer than its table row
            kv[1] = c.width * 16 + 1
        elif change == "pages":
            table[1, 2], table[1, 3] = 1 << 30, -7
        else:
            starts[2] = starts[1] - 1  # falling: the second sequence, and the third's start
        b = Z.KvBatch(starts, kv, table, T=c.T, max_q=c.max_q, max_kv=1 << 20)
        Z.kv_attend(c.cache, 0, b, c.q, out=out, err=err)
        assert int(err) == (Z.ERR_BAD_PAGE if change == "pages" else Z.ERR_BAD_SEQ)
        assert torch.equal(out[:c.starts[1]], good[:c.starts[1]])
        if change == "long":
            assert (out[mid] == 5).all() and torch.equal(out[c.starts[2]:], good[c.starts[2]:])
    with pytest.raises(Z.ZestError, match="error bits 0x8"):
        Z.kv_attend(c.cache, 0, Z.KvBatch(c.q_start, c.kv_len, c.table, T=c.T, max_q=c.max_q, max_kv=150), c.q)


def test_captured_replayed_and_beside_another_stream():
    """Two captured calls with a workspace each, replayed at once on two streams over changing lengths."""
    cs = [Case([(1, 4000), (1, 900)], 8, 2, 128, 16, BF, seed=11), Case([(33, 4000)], 8, 2, 128, 64, BF, seed=12)]
    calls = []
    for c in cs:
        out = torch.zeros_like(c.q)
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        ws = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            Z.kv_attend(c.cache, 0, c.batch, c.q, out=out, err=err, workspace=ws)
        st.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            Z.kv_attend(c.cache, 0, c.batch, c.q, out=out, err=err, workspace=ws)
        calls.append((c, out, err, ws, st, g))
    for shorter in (0, 300, 1500):
        for c, out, err, ws, st, g in calls:
            c.kv_len -= shorter * (c.kv_len > 2 * shorter).int()
            c.lens = list(zip([n for n, _ in c.lens], c.kv_len.tolist()))
        torch.cuda.synchronize()
        for _ in range(3):
            for c, out, err, ws, st, g in calls:
                with torch.cuda.stream(st):
                    g.replay()
        torch.cuda.synchronize()
        for c, out, err, ws, st, g in calls:
            assert int(err) == 0
            c.check(out)


@pytest.mark.parametrize("d,lens", [(128, [(1, 3000)]), (64, [(2, 5000), (1, 2000)]), (128, [(40, 6000)]),
                                    (256, [(30, 5000)])])
def test_a_row_with_a_part_that_never_came_stays(d, lens):
    """A block whose wait runs out marks its part of a row with a maximum of NaN. Such marks set by hand between the
    two kernels of a captured call, the first of them turned off: the join leaves those rows, and makes the others."""
    from cuda.bindings import runtime as rt

    c = Case(lens, 8, 2, d, 16, BF, seed=19)
    out, err = torch.zeros_like(c.q), torch.zeros(1, dtype=torch.int32, device="cuda")
    ws = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    Z.kv_attend(c.cache, 0, c.batch, c.q, out=out, err=err, workspace=ws)
    good = out.clone()
    c.check(good)
    g = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(g):
        Z.kv_attend(c.cache, 0, c.batch, c.q, out=out, err=err, workspace=ws)
    handle = rt.cudaGraph_t(g.raw_cuda_graph())
    n = rt.cudaGraphGetNodes(handle, 0)[2]
    assert n == 2, "the keys are cut: the attention, and the join of its parts"
    e, roots, _ = rt.cudaGraphGetRootNodes(handle, 1)
    assert int(e) == 0
    g.instantiate()
    assert int(rt.cudaGraphNodeSetEnabled(rt.cudaGraphExec_t(g.raw_cuda_graph_exec()), roots[0], 0)[0]) == 0
    ml = ws.view(torch.float32)
    rows, missing = c.T * c.heads, torch.zeros(c.T, c.heads, dtype=torch.bool, device="cuda")
    for part, t, head in ((0, 0, 1), (1, c.T - 1, 6)):
        ml[2 * (part * rows + t * c.heads + head)] = math.nan
        missing[t, head] = True
    out.fill_(5.0)
    g.replay()
    torch.cuda.synchronize()
    assert (out[missing] == 5).all() and torch.equal(out[~missing], good[~missing]) and int(err) == 0


def test_the_same_bits_every_time():
    c = Case([(1, 3000), (1, 50)], 8, 2, 128, 16, BF, seed=1)
    first = Z.kv_attend(c.cache, 0, c.batch, c.q)
    for _ in range(5):
        assert torch.equal(Z.kv_attend(c.cache, 0, c.batch, c.q), first)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_rows_past_the_last_move_no_bits(d):
    """A tile's rows past its tokens, or past its sequence's, hold what lay there: nothing of it shows."""
    c = Case([(50, 900), (45, 400)], 12, 2, d, 64, BF, seed=d)  # 6 heads a kv head: 126 of a tile's 128 rows
    first = Z.kv_attend(c.cache, 0, c.batch, c.q).clone()
    c.check(first)
    loud = Case([(128, 600)] * 8, 64, 4, d, 64, BF, seed=1)  # every row of every tile
    for gain in (300.0, 3e4):
        Z.kv_attend(loud.cache, 0, loud.batch, (loud.q.float() * gain).to(BF))
        assert torch.equal(Z.kv_attend(c.cache, 0, c.batch, c.q), first)
        q = c.q.clone()
        q[50:] = (q[50:].float() * gain).to(BF)
        assert torch.equal(Z.kv_attend(c.cache, 0, c.batch, q)[:50], first[:50])


@pytest.mark.parametrize("n_seqs,group", [(65535, 2), (4000, 24)])
def test_the_most_sequences(n_seqs, group):
    """65,535 of one token each, of 1 to 3 tokens in all; and as many tiles of a token's 24 heads."""
    d, g = 16, torch.Generator("cuda").manual_seed(3)
    k, v = (torch.randn(1, n_seqs, 16, 1, d, device="cuda", generator=g).to(BF) for _ in range(2))
    q = torch.randn(n_seqs, group, d, device="cuda", generator=g).to(BF)
    kv = (torch.arange(n_seqs, device="cuda") % 3 + 1).int()
    pages = torch.arange(n_seqs - 1, -1, -1, dtype=torch.int32, device="cuda")
    b = Z.KvBatch(torch.arange(n_seqs + 1, dtype=torch.int32, device="cuda"), kv, pages[:, None].contiguous(), T=n_seqs,
                  max_q=1, max_kv=3)
    kn, vn = (torch.randn(n_seqs, 1, d, device="cuda", generator=g) for _ in range(2))
    cache = Z.KvCache(k, v)
    Z.kv_append(cache, 0, b, kn, vn)
    at = (kv - 1).long()
    ks, vs = (x[0, pages.long(), :, 0] for x in (k, v))  # [n_seqs][16][d]
    rows = torch.arange(n_seqs, device="cuda")
    assert torch.equal(ks[rows, at], kn[:, 0].to(BF)) and torch.equal(vs[rows, at], vn[:, 0].to(BF))
    got = Z.kv_attend(cache, 0, b, q).double()
    z = torch.einsum("shd,sjd->shj", q.double(), ks[:, :3].double()) / 4
    z.masked_fill_(torch.arange(3, device="cuda") >= kv[:, None, None], -math.inf)
    p = torch.softmax(z, -1)
    want, mean = (torch.einsum("shj,sjd->shd", p, x) for x in (vs[:, :3].double(), vs[:, :3].double().abs()))
    assert bool(((got - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -11) * mean).all())


@pytest.mark.parametrize("n", [1, 200])
def test_offsets_past_32_bits(n):
    """A pool of more than 2^32 values whose sequences lie at its end."""
    pages, page, kv_heads, d = (1 << 32) // (64 * 8 * 128) + 40, 64, 8, 128
    k = torch.zeros(1, pages, page, kv_heads, d, dtype=BF, device="cuda")
    v = torch.zeros_like(k)
    small = Case([(n, 1500)], 32, kv_heads, d, page, BF, seed=13)
    rows = [pages - 1 - p for p in range(len(small.rows[0]))]
    for a, b in zip(small.rows[0], rows):
        k[0, b], v[0, b] = small.k[0, a], small.v[0, a]
    batch = Z.KvBatch(small.q_start, small.kv_len, i32([rows]), T=n, max_q=n, max_kv=1500)
    small.check(Z.kv_attend(Z.KvCache(k, v), 0, batch, small.q))
