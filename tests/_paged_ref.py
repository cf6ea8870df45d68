"""Plain 64-bit restatements of the paged cache's operators (test helper):
position by position, page by page, from the definitions in
include/m27b_paged.h."""
import math

import numpy as np

U = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}  # half a unit in the last place, relative: 8 and 11 significant bits


def cdiv(a, b):
    return -(-a // b)


def span(i, nq, nkv, window):
    """Positions [lo, hi) that new token i of nq sees, nkv positions cached."""
    hi = max(0, nkv - nq + i + 1)
    return (max(0, hi - window) if window > 0 else 0), hi


def rope_factors(n_pos, n_rot, theta, kind="none", factor=1.0, ctx=0, fast=32.0, slow=1.0, attn=0.0):
    """complex [n_pos, n_rot / 2]"""
    f = np.array([theta ** (-2.0 * j / n_rot) for j in range(n_rot // 2)])
    mul = 1.0
    if kind == "linear":
        f = f / factor
    if kind == "yarn":
        at = [n_rot * math.log(ctx / (2 * math.pi * b)) / (2 * math.log(theta)) for b in (fast, slow)]
        lo, hi = max(0, math.floor(at[0])), min(n_rot - 1, math.ceil(at[1]))
        r = np.clip((np.arange(n_rot // 2) - lo) / max(hi - lo, 0.001), 0, 1)
        f = f / factor * r + f * (1 - r)
        mul = attn if attn > 0 else 0.1 * math.log(factor) + 1
    return mul * np.exp(1j * np.arange(n_pos)[:, None] * f)


def norm_rope(x, w, eps, z, n_rot, interleaved):
    """x [..., hd] fp64 rotated by the factors z [n_rot / 2] (complex)."""
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    x = x.copy()
    a, b = (slice(0, n_rot, 2), slice(1, n_rot, 2)) if interleaved else (slice(0, n_rot // 2), slice(n_rot // 2, n_rot))
    t = (x[..., a] + 1j * x[..., b]) * z
    x[..., a], x[..., b] = t.real, t.imag
    return x


def attend(q, keys, vals, scale, window):
    """One sequence: q [nq, n_q, hd], keys / vals [nkv, n_kv, hd] fp64.  Returns
    out, lse, the absolute weighted values sum p |v|, and the largest
    scale * sum |q||k| of a row (the tolerances' scale)."""
    nq, n_q, hd = q.shape
    nkv, n_kv, _ = keys.shape
    out, lse = np.zeros((nq, n_q, hd)), np.full((nq, n_q), -np.inf)
    mag, big = np.zeros((nq, n_q, hd)), np.zeros((nq, n_q))
    for i in range(nq):
        lo, hi = span(i, nq, nkv, window)
        if hi <= lo:
            continue
        for h in range(n_q):
            j = h // (n_q // n_kv)
            s = scale * (keys[lo:hi, j] @ q[i, h])
            m = s.max()
            e = np.exp(s - m)
            p = e / e.sum()
            out[i, h] = p @ vals[lo:hi, j]
            lse[i, h] = m + math.log(e.sum())
            mag[i, h] = p @ np.abs(vals[lo:hi, j])
            big[i, h] = scale * (np.abs(keys[lo:hi, j]) @ np.abs(q[i, h])).max()
    return out, lse, mag, big


class Pages:
    """The page upkeep on lists; `data[plane][page]` any values."""

    def __init__(self, n_rows, n_cols, n_pages, ps, data):
        self.n_cols, self.ps, self.data = n_cols, ps, data
        self.table = [[-1] * n_cols for _ in range(n_rows)]
        self.ref, self.lens = [0] * n_pages, [0] * n_rows

    def free_pages(self):
        return [p for p, n in enumerate(self.ref) if n <= 0]

    def _move(self, pairs):
        for plane in self.data:
            old = [plane[a].copy() for a, _ in pairs]
            for (_, b), v in zip(pairs, old):
                plane[b] = v

    def resize(self, rows, lens):
        """None, or why the request is refused."""
        n, ps = len(self.lens), self.ps
        if any(not 0 <= r < n for r in rows) or len(set(rows)) < len(rows):
            return "bad"
        if any(x < 0 or cdiv(x, ps) > self.n_cols for x in lens):
            return "bad"
        plan, need = [], 0
        for r, x in zip(rows, lens):
            old = self.lens[r]
            own = x > old and old % ps and self.ref[self.table[r][old // ps]] > 1
            k = max(0, cdiv(x, ps) - cdiv(old, ps)) + bool(own)
            plan.append((own, k))
            need += k
        free = self.free_pages()
        if need > len(free):
            return "full"
        take, pairs, drops = iter(free), [], []
        for (r, x), (own, k) in zip(zip(rows, lens), plan):
            old = self.lens[r]
            if own:
                p, new = self.table[r][old // self.ps], next(take)
                pairs.append((p, new))
                drops.append(p)
                self.table[r][old // self.ps] = new
                self.ref[new] = 1
            for c in range(cdiv(old, ps), cdiv(x, ps)):
                self.table[r][c] = next(take)
                self.ref[self.table[r][c]] = 1
            for c in range(cdiv(x, ps), cdiv(old, ps)):
                drops.append(self.table[r][c])
                self.table[r][c] = -1
            self.lens[r] = x
        for p in drops:
            self.ref[p] -= 1
        self._move(pairs)

    def fork(self, src, dst):
        n, ps = len(self.lens), self.ps
        if any(not 0 <= r < n for r in src + dst) or len(set(dst)) < len(dst) or set(src) & set(dst):
            return "bad"
        if any(self.lens[d] for d in dst):
            return "bad"
        free = self.free_pages()
        if sum(self.lens[s] % ps != 0 for s in src) > len(free):
            return "full"
        take, pairs = iter(free), []
        for s, d in zip(src, dst):
            for c in range(cdiv(self.lens[s], ps)):
                p = self.table[s][c]
                if (c + 1) * ps > self.lens[s]:
                    new = next(take)
                    pairs.append((p, new))
                    p = new
                self.table[d][c] = p
                self.ref[p] += 1
            self.lens[d] = self.lens[s]
        self._move(pairs)

    def free(self, rows):
        for r in rows:
            for c in range(cdiv(self.lens[r], self.ps)):
                self.ref[self.table[r][c]] -= 1
                self.table[r][c] = -1
            self.lens[r] = 0

    def compact(self):
        live = sum(n > 0 for n in self.ref)
        src = [p for p in range(live, len(self.ref)) if self.ref[p] > 0]
        dst = [p for p in range(live) if self.ref[p] <= 0]
        to = dict(zip(src, dst))
        for a, b in to.items():
            self.ref[b], self.ref[a] = self.ref[a], 0
        self.table = [[to.get(p, p) for p in r] for r in self.table]
        self._move(list(to.items()))
        return live
