"""A plain model of the 4-bit cache for the tests: page bookkeeping in Python,
rows and attention in 64-bit numpy, written from the definitions."""
from __future__ import annotations

import math

import numpy as np

TILE = 32
STEP = 0.3352


def rotation(signs):
    """R as a 64-bit matrix, y = R x."""
    d = signs.shape[1]
    h = np.ones((1, 1))
    while h.shape[0] < d:
        h = np.block([[h, h], [h, -h]])
    r = np.eye(d)
    for s in signs:
        r = (h * s) @ r / math.sqrt(d)
    return r


def quantise(x, r):
    """64-bit codes' levels, scales, and how far each value is from a step's edge."""
    y = x.astype(np.float64) @ r.T
    sq = (y * y).sum(-1, keepdims=True)
    with np.errstate(divide="ignore", invalid="ignore"):
        z = np.where(sq > 0, y / (STEP * np.sqrt(sq / y.shape[-1])), 0.0)
        level = np.clip(np.floor(z), -8, 7) + 0.5
        scale = np.where(sq > 0, sq / (level * y).sum(-1, keepdims=True), 0.0)
    edge = np.where((z > -8.5) & (z < 7.5), np.abs(z - np.rint(z)), 1.0)
    return level, scale[..., 0], edge


def unpack(tiles, d):
    """(levels, scales) of keys and of values of tiles [..., 32 (d + 8)]."""
    lead, half = tiles.shape[:-1], TILE * (d // 2)

    def levels(c):
        return np.stack((c & 15, c >> 4), -1).reshape(*c.shape[:-1], d).astype(np.float64) - 7.5

    def floats(b):
        return np.ascontiguousarray(b).view(np.float32).astype(np.float64)

    k = tiles[..., :half].reshape(*lead, TILE, d // 2)
    at = half + 4 * TILE
    v = np.swapaxes(tiles[..., at:at + half].reshape(*lead, TILE // 2, d // 4, 2, 2), -2, -3)
    v = np.ascontiguousarray(v).reshape(*lead, TILE, d // 2)
    return ((levels(k), floats(tiles[..., half:at])),
            (levels(v), floats(tiles[..., at + half:])))


def held(pool, table_row, n, d):
    """Rotated keys and values [heads, n, d] of a sequence of n tokens in one
    layer's pool [pages, heads, tiles, bytes], with their levels and scales."""
    pages = pool.shape[2] * TILE
    tiles = pool[table_row[:-(-n // pages)]].transpose(1, 0, 2, 3)
    out = []
    for level, scale in unpack(tiles, d):
        h = level.shape[0]
        out.append((level.reshape(h, -1, d)[:, :n], scale.reshape(h, -1)[:, :n]))
    return out


def attend(q, kv, r, scale):
    """Reference and error scale of one sequence: q [rows, q_heads, d] are the
    last rows of n tokens.  Returns out, lse, the weighted sum of |v| as a norm
    (rotated), and the largest sum |q_i k_i| of a row, all per (row, head)."""
    (kl, ks), (vl, vs) = kv
    with np.errstate(invalid="ignore", over="ignore"):
        k, v = kl * ks[..., None], vl * vs[..., None]
    rows, hq, d = q.shape
    n, group = k.shape[1], hq // k.shape[0]
    y = q.astype(np.float64) @ r.T
    out, lse = np.zeros((rows, hq, d)), np.full((rows, hq), -np.inf)
    size, reach = np.zeros((rows, hq)), np.zeros((rows, hq))
    for i in range(rows):
        m = n - rows + i + 1
        if m <= 0:
            continue
        for h in range(hq):
            e = k[h // group, :m] @ y[i, h] * scale
            top = e.max()
            p = np.exp(e - top)
            lse[i, h] = top + np.log(p.sum())
            p /= p.sum()
            out[i, h] = (p @ v[h // group, :m]) @ r
            size[i, h] = np.linalg.norm(p @ np.abs(v[h // group, :m]))
            reach[i, h] = (np.abs(k[h // group, :m]) @ np.abs(y[i, h])).max() * scale
    return out, lse, size, reach


def prompt(q, k, v, causal, scale):
    """out, lse, sum p |v| and the largest sum |q_i k_i| of one sequence."""
    q, k, v = (x.astype(np.float64) for x in (q, k, v))
    rows, hq, d = q.shape
    n, group = k.shape[0], hq // k.shape[1]
    out, lse = np.zeros((rows, hq, d)), np.full((rows, hq), -np.inf)
    size, reach = np.zeros((rows, hq, d)), np.zeros((rows, hq))
    for i in range(rows):
        m = min(n, i + n - rows + 1) if causal else n
        if m <= 0:
            continue
        for h in range(hq):
            kk, vv = k[:m, h // group], v[:m, h // group]
            e = kk @ q[i, h] * scale
            top = e.max()
            p = np.exp(e - top)
            lse[i, h] = top + np.log(p.sum())
            p /= p.sum()
            out[i, h], size[i, h] = p @ vv, p @ np.abs(vv)
            reach[i, h] = (np.abs(kk) @ np.abs(q[i, h])).max() * scale
    return out, lse, size, reach


class Pages:
    """The bookkeeping: lowest free pages first, in the list's order."""

    def __init__(self, n_pages, max_seqs, max_pages, page):
        self.refs = np.zeros(n_pages, np.int32)
        self.table = np.full((max_seqs, max_pages), -1, np.int32)
        self.lens = np.zeros(max_seqs, np.int32)
        self.page = page
        self.moves = []  # (from, to) of the last call

    def pages(self, n):
        return -(-int(n) // self.page)

    def _take(self, n):
        p = np.flatnonzero(self.refs == 0)[:n]
        self.refs[p] = 1
        return list(p)

    def extend(self, seqs, counts):
        self.moves, plan = [], []
        for s, c in zip(seqs, counts):
            have, n = self.pages(self.lens[s]), int(self.lens[s])
            cow = c > 0 and n % self.page and self.refs[self.table[s, have - 1]] > 1
            plan.append((s, c, have, bool(cow)))
        need = sum(self.pages(self.lens[s] + c) - have + cow for s, c, have, cow in plan)
        if need > (self.refs == 0).sum():
            return False
        drop = []
        for s, c, have, cow in plan:
            fresh = self._take(self.pages(self.lens[s] + c) - have + cow)
            if cow:
                self.moves.append((int(self.table[s, have - 1]), int(fresh[0])))
                drop.append(self.table[s, have - 1])
            self.table[s, have - cow:have - cow + len(fresh)] = fresh
            self.lens[s] += c
        for p in drop:
            self.refs[p] -= 1
        return True

    def fork(self, src, dst, lens=None):
        for i, (a, b) in enumerate(zip(src, dst)):
            n = self.lens[a] if lens is None else min(self.lens[a], lens[i])
            m = self.pages(n)
            self.table[b, :m] = self.table[a, :m]
            self.refs[self.table[a, :m]] += 1
            self.lens[b] = n

    def copy(self, src, dst):
        self.moves = []
        for a, b in zip(src, dst):
            m = self.pages(self.lens[a])
            fresh = self._take(m)
            self.moves += [(int(x), int(y)) for x, y in zip(self.table[a, :m], fresh)]
            self.table[b, :m] = fresh
            self.lens[b] = self.lens[a]

    def truncate(self, seqs, lens=None):
        for i, s in enumerate(seqs):
            n = min(self.lens[s], 0 if lens is None else lens[i])
            a, b = self.pages(n), self.pages(self.lens[s])
            for p in self.table[s, a:b]:
                self.refs[p] -= 1
            self.table[s, a:b] = -1
            self.lens[s] = n

    def compact(self):
        used = self.refs > 0
        n = int(used.sum())
        high, low = np.flatnonzero(used[n:]) + n, np.flatnonzero(~used[:n])
        self.moves = list(zip(high.tolist(), low.tolist()))
        to = np.arange(len(used), dtype=np.int32)
        to[high] = low
        self.refs[low] = self.refs[high]
        self.refs[high] = 0
        self.table = np.where(self.table >= 0, to[np.maximum(self.table, 0)], -1).astype(np.int32)
