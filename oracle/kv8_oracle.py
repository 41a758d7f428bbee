"""Plain numpy restatement of the rotary positions and the 8-bit KV cache.

Values, scores and softmax sums are in 64 bits.  Where the definition rounds
(codes and scales), the same 32-bit products and quotients are formed, so that
codes can be compared bit for bit.
"""

import math

import numpy as np

F = np.float32
QMAX = {"int8": 127.0, "e4m3": 448.0}
TINY = F(2.0 ** -100)


def e4m3_round(x):
    """Nearest value of e4m3 (ties to even, largest magnitude 448)."""
    x = np.asarray(x, np.float64)
    _, e = np.frexp(x)
    q = np.ldexp(1.0, np.maximum(e - 1, -6) - 3)
    return np.clip(np.rint(x / q) * q, -448.0, 448.0)


def encode(x, code):
    """Codes, as the numbers that they stand for before the scale."""
    x = np.asarray(x, np.float64)
    return np.clip(np.rint(x), -127, 127) if code == "int8" else e4m3_round(x)


def scale_of(rows, code):
    """float32 scale of a group's rows [n, D]."""
    a = np.abs(np.asarray(rows, F))
    if not np.isfinite(a).all():
        return F(np.nan)
    m = a.max(initial=F(0))
    return F(0) if m < TINY else F(m * F(1.0 / QMAX[code]))


def rotary(x, positions, inv_freq, sections, interleaved=False, inverse=False):
    """x [T, H, D] float64; positions [T, axes]; inv_freq float32 [rot / 2]."""
    axis = np.repeat(np.arange(len(sections)), sections)
    a = positions[:, axis].astype(np.float64) * inv_freq.astype(np.float64)
    z = np.exp(1j * (-a if inverse else a))[:, None, :]
    rot = 2 * len(axis)
    y = np.array(x, np.float64)
    i = np.arange(rot // 2)
    p, q = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    w = (y[..., p] + 1j * y[..., q]) * z
    y[..., p], y[..., q] = w.real, w.imag
    return y


class Cache:
    """codes [nb, H, P, D] and scales [nb, H, P / group], K and V."""

    def __init__(self, code, codes, scales, table, group):
        self.code, self.codes, self.scales, self.table, self.group = code, codes, scales, table, group
        self.nb, self.H, self.P, self.D = codes[0].shape

    def at(self, s, r):
        """(page, row) of a sequence's row r, or None outside the table or the cache."""
        if r < 0 or r // self.P >= self.table.shape[1]:
            return None
        page = int(self.table[s, r // self.P])
        return (page, r % self.P) if 0 <= page < self.nb else None

    def values(self, w, s, h, n):
        """Rows [0, n) as float64 values; rows that cannot be reached are zeros."""
        out = np.zeros((n, self.D))
        for r in range(n):
            a = self.at(s, r)
            if a is not None:
                out[r] = self.codes[w][a[0], h, a[1]].astype(np.float64) * np.float64(
                    self.scales[w][a[0], h, a[1] // self.group])
        return out

    def write(self, w, x, starts, cu):
        """x [T, H, D] float32."""
        g = self.group
        for s, start in enumerate(starts):
            rows = x[cu[s]:cu[s + 1]]
            if not len(rows):
                continue
            end = start + len(rows)
            for first in range(start // g * g, end, g):
                a = self.at(s, first)
                if a is None:
                    continue
                lo, hi = max(first, start), min(first + g, end)
                for h in range(self.H):
                    new = np.asarray(rows[lo - start:hi - start, h], F)
                    want, sc = scale_of(new, self.code), self.scales[w]
                    gi = (a[0], h, a[1] // g)
                    was, now = sc[gi], want
                    if lo > first:
                        now = F(np.nan) if np.isnan(was) or np.isnan(want) else max(was, want)
                        if was < now:
                            old = self.codes[w][a[0], h, a[1]:a[1] + lo - first]
                            old[...] = encode(np.asarray(old, F) * F(was / now), self.code)
                    sc[gi] = now
                    q = np.zeros_like(new) if not now > 0 else encode(new * F(F(1) / now), self.code)
                    self.codes[w][a[0], h, a[1] + lo - first:a[1] + hi - first] = q

    def attend(self, q, lens, softcap=0.0, width=None):
        """q [B, Lq, Hq, D] float64 -> (out, lse, weights, bound): float64; bound
        [B, Lq, Hq] is the largest sum of |q k| scale over a row's keys."""
        B, Lq, Hq, D = q.shape
        G = Hq // self.H
        out, lse = np.zeros(q.shape), np.full((B, Lq, Hq), -np.inf)
        width = self.table.shape[1] * self.P if width is None else width
        weights, size = np.zeros((B, self.H, width)), np.zeros((B, Lq, Hq))
        mass = np.zeros(q.shape)
        for s in range(B):
            n = max(0, min(int(lens[s]), self.table.shape[1] * self.P))
            for h in range(self.H):
                k, v = self.values(0, s, h, n), self.values(1, s, h, n)
                for i in range(Lq):
                    m = n - Lq + 1 + i
                    if m <= 0:
                        continue
                    for j in range(h * G, (h + 1) * G):
                        z = k[:m] @ q[s, i, j] / math.sqrt(D)
                        size[s, i, j] = (np.abs(k[:m]) @ np.abs(q[s, i, j])).max() / math.sqrt(D)
                        if softcap:
                            z = softcap * np.tanh(z / softcap)
                        top = z.max()
                        e = np.exp(z - top)
                        lse[s, i, j] = top + np.log(e.sum())
                        p = e / e.sum()
                        out[s, i, j] = p @ v[:m]
                        mass[s, i, j] = p @ np.abs(v[:m])
                        weights[s, h, :min(m, width)] += p[:width]
        return out, lse, weights, size, mass

    def evict(self, lens, weights, budget, recent):
        """In place, weights [B, H, W] float32 too; rows past W weigh 0.  Returns (kept, new_lens)."""
        B, H, W = weights.shape
        rows = self.table.shape[1] * self.P
        kept = np.full((B, H, budget), -1, np.int32)
        new = np.zeros(B, np.int32)
        for s in range(B):
            n = max(0, min(int(lens[s]), rows))
            m = new[s] = min(n, budget)
            for h in range(H):
                idx, held = np.arange(n), np.zeros(max(rows, W), F)
                held[:W] = weights[s, h]
                if n > budget:
                    w = held[:n - recent].astype(np.float64)
                    w = np.where(np.isnan(w), np.inf, w), np.isnan(w)
                    order = np.lexsort((np.arange(n - recent), -w[0], ~w[1]))
                    idx = np.sort(np.concatenate([order[:budget - recent], np.arange(n - recent, n)])).astype(int)
                kept[s, h, :m] = idx
                if n <= budget:
                    continue
                held[:m], held[m:n] = held[idx], 0
                weights[s, h] = held[:W]
                for w in (0, 1):
                    self._move(w, s, h, idx)
        return kept, new

    def _move(self, w, s, h, idx):
        g = self.group
        src = [self.at(s, int(r)) for r in idx]
        codes = np.stack([self.codes[w][a[0], h, a[1]].copy() if a else np.zeros(self.D, F) for a in src])
        scales = np.array([self.scales[w][a[0], h, a[1] // g] if a else 0 for a in src], F)
        for j0 in range(0, len(idx), g):
            a = self.at(s, j0)
            if a is None:
                continue
            big = F(np.nan) if np.isnan(scales[j0:j0 + g]).any() else scales[j0:j0 + g].max()
            self.scales[w][a[0], h, a[1] // g] = big
            for j in range(j0, min(j0 + g, len(idx))):
                q = codes[j]
                if scales[j] < big:
                    q = encode(np.asarray(q, F) * F(scales[j] / big), self.code)
                self.codes[w][a[0], h, a[1] + j - j0] = q
