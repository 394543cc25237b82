"""The paged cache's operators in plain 64-bit form, for the tests: the
attention and the rotation by their definitions, the page operations page by
page on host lists."""
import math

import torch


def laid_out(pool, row, n, page):
    """The first n tokens of one layer's pool [pages][page][heads][d] along a table row, in 64 bits."""
    pages = [pool[int(row[j])] for j in range(-(-n // page))]
    return torch.cat(pages)[:n].double() if pages else pool.new_zeros((0,) + pool.shape[2:]).double()


def attention(q, k, v, first, scale, causal, window):
    """q [n][H][d], k and v [S][Hk][d] in 64 bits, the first row at position `first`. Returns the result, and the
    mean of |v| under the same weights (what a rounding of the weights can move), and the keys a row sees."""
    n, H, d = q.shape
    S, Hk = k.shape[:2]
    pos = first + torch.arange(n, device=q.device)[:, None]
    j = torch.arange(S, device=q.device)[None]
    sees = torch.ones(n, S, dtype=torch.bool, device=q.device)
    if causal:
        sees &= j <= pos
    if window:
        sees &= j > pos - window
    o, a = torch.zeros_like(q), torch.zeros_like(q)
    for h in range(H):
        g = h // (H // Hk)
        z = torch.where(sees, q[:, h] @ k[:, g].T * scale, -math.inf)
        top = z.amax(-1, keepdim=True) if S else z.new_zeros(n, 1)
        p = torch.exp(z - torch.where(top == -math.inf, 0.0, top))
        # weights of keys that are not seen are zero whatever the value is
        p = torch.where(sees, p, 0.0)
        total = p.sum(-1, keepdim=True)
        p = p / torch.where(total == 0, 1.0, total)
        if torch.isfinite(v[:, g]).all():
            o[:, h], a[:, h] = p @ v[:, g], p @ v[:, g].abs()
        else:
            for i in range(n):
                w, x = p[i][sees[i]], v[sees[i], g]
                o[i, h], a[i, h] = (w[:, None] * x).sum(0), (w[:, None] * x.abs()).sum(0)
    return o, a, sees.sum(-1)


def turned(x, w, eps, rope, neox):
    """[T][heads][d] in 64 bits after the norm (eps >= 0), its weight, and the rotation by [T][n_dims]."""
    x = x.double()
    if eps >= 0:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
        if w is not None:
            x = x * w.double()
    if rope is None:
        return x
    cs, n = rope.double(), rope.shape[1]
    y = x.clone()
    for p in range(n // 2):
        i, j = (p, p + n // 2) if neox else (2 * p, 2 * p + 1)
        c, s = cs[:, 2 * p, None], cs[:, 2 * p + 1, None]
        y[..., i] = x[..., i] * c - x[..., j] * s
        y[..., j] = x[..., i] * s + x[..., j] * c
    return y


class Pages:
    """The page tables on the host, and which page's bytes each operation copies where."""

    def __init__(self, pages, seqs, width, page):
        self.refs, self.len = [0] * pages, [0] * seqs
        self.table = [[-1] * width for _ in range(seqs)]
        self.page = page

    def _held(self, n):
        return -(-n // self.page)

    def _take(self):
        p = self.refs.index(0)
        self.refs[p] = 1
        return p

    def grow(self, seq, add):
        for s, a in zip(seq, add):
            for j in range(self._held(self.len[s]), self._held(self.len[s] + a)):
                self.table[s][j] = self._take()
            self.len[s] += a
        return []

    def fork(self, src, dst):
        moves = []
        for a, b in zip(src, dst):
            n = self.len[a]
            if a == b:
                continue
            self.table[b] = [-1] * len(self.table[b])
            for j in range(self._held(n)):
                if (j + 1) * self.page <= n:
                    self.table[b][j] = self.table[a][j]
                    self.refs[self.table[a][j]] += 1
                else:
                    self.table[b][j] = self._take()
                    moves.append((self.table[a][j], self.table[b][j]))
            self.len[b] = n
        return moves

    def free(self, seq):
        for s in seq:
            for p in self.table[s]:
                if p >= 0:
                    self.refs[p] -= 1
            self.table[s], self.len[s] = [-1] * len(self.table[s]), 0
        return []

    def compact(self):
        live = sum(r != 0 for r in self.refs)
        high = [p for p in range(live, len(self.refs)) if self.refs[p]]
        moves = list(zip(high, [p for p in range(live) if not self.refs[p]]))
        for a, b in moves:
            self.refs[a], self.refs[b] = 0, self.refs[a]
        to = dict(moves)
        self.table = [[to.get(p, p) for p in row] for row in self.table]
        return moves
