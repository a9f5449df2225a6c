"""Plain restatements of the paged cache's operators for the tests: page bookkeeping one row after the other on
lists, attention and rotation in NumPy, in 64 bits where they are compared with a tolerance."""
import numpy as np


class Pages:
    """Table and counts as Python lists, with the operations done entry by entry."""

    def __init__(self, table, refs, page_size):
        self.table, self.refs, self.ps = [list(map(int, r)) for r in table], list(map(int, refs)), page_size

    def fork(self, parent):
        old = [list(r) for r in self.table]
        for b, p in enumerate(parent):
            if not -1 <= p < len(old):
                continue
            for j, was in enumerate(old[b]):
                now = -1 if p < 0 else old[p][j]
                self.table[b][j] = now
                for e, d in ((was, -1), (now, 1)):
                    if 0 <= e < len(self.refs):
                        self.refs[e] += d

    def reserve(self, rows):
        """rows: (sequence, position) each, position -1: idle.  Returns (pairs, failed, taken)."""
        pairs, failed, taken = [], 0, 0
        free = [p for p, r in enumerate(self.refs) if r <= 0]
        done = set()
        for s, pos in rows:
            if pos < 0 or (s, pos // self.ps) in done:
                continue
            j = pos // self.ps
            done.add((s, j))
            p = self.table[s][j]
            has = 0 <= p < len(self.refs)
            if has and self.refs[p] <= 1:
                continue
            if not free:
                failed += 1
                continue
            n = free.pop(0)
            taken += 1
            self.refs[n] = 1
            self.table[s][j] = n
            if has:
                self.refs[p] -= 1
                pairs.append((p, n))
        return pairs, failed, taken

    def compact(self, most):
        """Returns (pairs, pages in use, 1 + the highest page in use)."""
        pairs = []
        while len(pairs) < most:
            live = [p for p, r in enumerate(self.refs) if r > 0]
            free = [p for p, r in enumerate(self.refs) if r <= 0]
            if not live or not free or free[0] > live[-1]:
                break
            a, b = live[-1], free[0]
            pairs.append((a, b))
            self.refs[a], self.refs[b] = 0, self.refs[a]
            self.table = [[b if e == a else e for e in r] for r in self.table]
        live = [p for p, r in enumerate(self.refs) if r > 0]
        return pairs, len(live), (live[-1] + 1 if live else 0)


def rotate(x, cs, interleaved=True):
    """x [heads][hd] fp32 by (cos, sin) pairs cs [hd/2][2] in fp32, products and sums rounded one by one."""
    x, c, s = np.asarray(x, np.float32), np.float32(cs[:, 0]), np.float32(cs[:, 1])
    h = x.shape[1] // 2
    a, b = (x[:, 0::2], x[:, 1::2]) if interleaved else (x[:, :h], x[:, h:])
    ra, rb = a * c - b * s, a * s + b * c
    out = np.empty_like(x)
    if interleaved:
        out[:, 0::2], out[:, 1::2] = ra, rb
    else:
        out[:, :h], out[:, h:] = ra, rb
    return out


def attention(q, k, v, scale):
    """One row: q [heads][hd], k, v [positions][kv heads][hd]; 64-bit result and a bound on the error of an fp32
    evaluation of it.

    The bound: a score is a sum of hd products whose factors carry 22 bits or more, so it is off by at most
    d = |scale| (hd 2^-23 sum|q k| + 2^-21 max|q| sum|k|); a weight by a factor e^(2 d) and a few roundings, and a
    sum over n positions by n 2^-24 of its absolute sum, however it is ordered.  Twice that for the quotient."""
    q, k, v = (np.asarray(t, np.float64) for t in (q, k, v))
    g = q.shape[0] // k.shape[1]
    out, tol = np.zeros_like(q), np.zeros_like(q)
    for h in range(q.shape[0]):
        kk, vv = k[:, h // g], v[:, h // g]
        if not len(kk):
            continue
        s = kk @ q[h] * scale
        p = np.exp(s - s.max())
        p /= p.sum()
        d = abs(scale) * (q.shape[1] * 2.0 ** -23 * np.abs(kk * q[h]).sum(1)
                          + 2.0 ** -21 * np.abs(q[h]).max() * np.abs(kk).sum(1)).max()
        out[h] = p @ vv
        tol[h] = (p @ np.abs(vv)) * 2.0 * (2.0 * d + (len(kk) + 16) * 2.0 ** -24)
    return out, tol
