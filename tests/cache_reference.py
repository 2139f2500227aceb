"""A KV cache in pages, kept with Python lists and 64-bit values: what fa2_custom_mask's PagedCache4 has to agree with."""
import math

import numpy as np
import torch

PAGE = 64
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
LARGEST = {torch.float16: 13, torch.bfloat16: 125}        # exponent of a scale: 6 times it is finite in the type
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def stands_for(x, dtype):
    """The values [..., D] (D a multiple of 32, 64-bit) that x is kept as: 32 share the smallest power of two of which the largest magnitude is
    less than 7 times as large; each is the nearest magnitude, of two equally near ones the one of even index."""
    x = np.asarray(x, dtype=np.float64)
    groups = x.reshape(-1, 32)
    out = np.empty_like(groups)
    m = np.array(MAGNITUDES)
    top = np.abs(groups).max(axis=1)
    finite = np.isfinite(groups).all(axis=1)
    with np.errstate(all="ignore"):
        _, e = np.frexp(np.where(finite & (top > 0), top, 1.0))          # top in [2^(e-1), 2^e)
        e = e - 3
        e = np.where(top >= 7 * np.ldexp(1.0, e), e + 1, e)
        e = np.where(top > 0, np.clip(e, -127, LARGEST[dtype]), -127)
        y = np.abs(groups) / np.ldexp(1.0, e)[:, None]
        i = np.searchsorted(m, y, side="right").clip(1, 7)              # m[i - 1] <= y < m[i], or beyond the last
        mid = (m[i - 1] + m[i]) / 2
        up = np.where(i == 8, False, (y > mid) | ((y == mid) & (i % 2 == 0)))
        out = np.copysign(np.where(up, m[i], m[i - 1]), groups) * np.ldexp(1.0, e)[:, None]
    out[~finite] = np.nan
    return out.reshape(x.shape)


class Reference:
    def __init__(self, pages, heads, head_dim, sequences, tokens, dtype):
        self.P, self.H, self.D, self.S, self.M, self.dtype = pages, heads, head_dim, sequences, -(-tokens // PAGE), dtype
        D = max(64, head_dim)
        self.k, self.v = [np.full((pages, heads, PAGE, D), np.nan) for _ in range(2)]
        self.table, self.length, self.refs = [[] for _ in range(sequences)], [0] * sequences, [0] * pages

    def _padded(self, x):
        x = x.double().cpu().numpy()
        return np.pad(x, [(0, 0)] * (x.ndim - 1) + [(0, max(64, self.D) - self.D)])

    def append(self, k, v, at=None, counts=None, sequences=None):
        """Returns the words of the status that the call sets."""
        B, _, N, _ = k.shape
        k, v = [stands_for(self._padded(x), self.dtype) for x in (k, v)]
        said, held = set(), list(self.refs)
        free = [p for p in range(self.P) if self.refs[p] == 0]
        full = False
        done, given = [], []
        for b in range(B):
            s = b if sequences is None else sequences[b]
            n = N if counts is None else counts[b]
            if not 0 <= s < self.S or s in done:
                said.add(0)
                continue
            done.append(s)
            a = self.length[s] if at is None else at[b]
            if not 0 <= n <= N or not 0 <= a <= self.length[s] or a + n > self.M * PAGE:
                said.add(0)
                continue
            row = self.table[s]
            touched = range(a // PAGE, -(-(a + n) // PAGE)) if n else range(0)
            need = [j for j in touched if j >= len(row) or held[row[j]] > 1]
            if need and (full or len(need) > len(free)):
                full = True
                said.add(1)
                continue
            new = list(row[:-(-(a + n) // PAGE)])
            given += row[-(-(a + n) // PAGE):]
            for j in need:
                p = free.pop(0)
                if j < len(row):
                    given.append(row[j])
                    if j == a // PAGE:
                        self.k[p, :, :a % PAGE], self.v[p, :, :a % PAGE] = self.k[row[j], :, :a % PAGE], self.v[row[j], :, :a % PAGE]
                    new[j] = p
                else:
                    new.append(p)
                self.refs[p] = 1
            self.table[s], self.length[s] = new, a + n
            for i in range(n):
                p, t = new[(a + i) // PAGE], (a + i) % PAGE
                self.k[p, :, t], self.v[p, :, t] = k[b, :, i], v[b, :, i]
        for p in given:
            self.refs[p] -= 1
        return said

    def values(self, s, begin=0, end=None):
        """(k, v) [heads, tokens, head_dim] of a sequence."""
        end = self.length[s] if end is None else end
        t = np.arange(begin, end)
        page = np.array(self.table[s] + [0], dtype=int)[t // PAGE] if len(t) else np.zeros(0, dtype=int)
        return [np.moveaxis(x[page, :, t % PAGE], 0, 1)[..., :self.D] for x in (self.k, self.v)]

    def read(self, tokens, start=None, sequences=None):
        rows = range(self.S) if sequences is None else sequences
        k, v = [np.zeros((len(rows), self.H, tokens, self.D)) for _ in range(2)]
        for b, s in enumerate(rows):
            a = 0 if start is None else start[b]
            lo, hi = max(0, a), min(self.length[s], a + tokens)
            if hi > lo:
                k[b, :, lo - a:hi - a], v[b, :, lo - a:hi - a] = self.values(s, lo, hi)
        return k, v

    def fork(self, parents, children):
        said = set()
        for i, (p, c) in enumerate(zip(parents, children)):
            if not (0 <= p < self.S and 0 <= c < self.S) or p in children or c in children[:i] or self.length[c]:
                said.add(0)
                continue
            self.table[c], self.length[c] = list(self.table[p]), self.length[p]
            for x in self.table[p]:
                self.refs[x] += 1
        return said

    def free(self, sequences=None, keep=None):
        said, done = set(), []
        for i, s in enumerate(range(self.S) if sequences is None else sequences):
            n = 0 if keep is None else keep[i]
            again = s in done
            done.append(s)
            if not 0 <= s < self.S or n < 0 or again:
                said.add(0)
            elif n < self.length[s]:
                for p in self.table[s][-(-n // PAGE):]:
                    self.refs[p] -= 1
                self.table[s], self.length[s] = self.table[s][:-(-n // PAGE)], n
        return said

    def compact(self):
        U = sum(r > 0 for r in self.refs)
        holes, movers = [p for p in range(U) if not self.refs[p]], [p for p in range(U, self.P) if self.refs[p]]
        for h, m in zip(holes, movers):
            self.k[h], self.v[h] = self.k[m], self.v[m]
            self.refs[h], self.refs[m] = self.refs[m], 0
            self.table = [[h if p == m else p for p in row] for row in self.table]

    def tables(self):
        return [row + [-1] * (self.M - len(row)) for row in self.table]


def attention(q, k, v, first, scale, kept=None):
    """One sequence in 64 bits: q [H, n, D], k, v [heads, T, D], query i at position first + i; kept: bool [H, n, pages] or None.
    Returns o [H, n, D], lse [H, n], and the softmax's mean of |v| (for bounds of rounding errors).  A value that is not a number counts
    where its token is seen."""
    H, n, D = q.shape
    heads, T = k.shape[:2]
    o, a, lse = np.zeros((H, n, D)), np.zeros((H, n, D)), np.full((H, n), -np.inf)
    t = np.arange(T)
    with np.errstate(all="ignore"):
        for h in range(H):
            for i in range(n):
                see = t <= first + i
                if kept is not None:
                    see = see & kept[h, i][t // PAGE]
                if not see.any():
                    continue
                kk, vv = k[h // (H // heads)][see], v[h // (H // heads)][see]
                s = (kk * q[h, i]).sum(-1) * scale
                m = s.max()
                p = np.exp(s - m)
                o[h, i], a[h, i], lse[h, i] = p @ vv / p.sum(), p @ np.abs(vv) / p.sum(), m + np.log(p.sum())
    return o, lse, a


def within(o, ref, mean, dtype, out=None):
    """|o - ref| within the roundings of P (half a step of the type of the products, relative, each: half a step of the mean of |v| together) and
    of the result (half a step of it), and 2^-12 of the mean of |v| for the sums and exponentials in 32 bits (scores of up to 100: their
    errors of up to 128 * 2^-24 * 100 are those of the numerators' logarithms)."""
    o = o.double().cpu().numpy() if isinstance(o, torch.Tensor) else o
    bound = HALF_STEP[dtype] * mean + HALF_STEP[out or dtype] * (np.abs(ref) + HALF_STEP[dtype] * mean) + 2.0 ** -12 * mean + 2.0 ** -25
    bad = np.isnan(ref)
    return bool(np.array_equal(np.isnan(o), bad)) and bool((np.abs(o - ref)[~bad] <= bound[~bad]).all())


def scale_of(D):
    return 1.0 / math.sqrt(D)
