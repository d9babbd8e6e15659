"""The 4-bit latent records and the page tables in plain numpy, values in 64 bits (test infrastructure; nothing here is on a product
path).  The layout is that of include/dsa_b200.h."""
import numpy as np

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
SIGN = (15, 12, 9, 14)
NUMBER = ((8, 7, 6), (5, 4, 3), (2, 1, 0), (11, 10, 13))
SCALES = np.array([(8 + m) * 2.0 ** (e - 18) for e in range(31) for m in range(8)])       # by byte
PAGE = 64


def nearest(values, grid):
    """Index of the grid value nearest to each value, ties to the even index."""
    up = np.clip(np.searchsorted(grid, values), 0, len(grid) - 1)
    dn = np.maximum(up - 1, 0)
    a, b = values - grid[dn], grid[up] - values
    return np.where((a < b) | ((a == b) & (dn % 2 == 0)), dn, up)


def encode(kv):
    """Rows [N, 576] float64 -> (numbers [N, 512], signs [N, 512], scale bytes [N, 32], rope [N, 64])."""
    lat = kv[:, :512].reshape(-1, 32, 16)
    bad = ~np.isfinite(lat).all(-1)
    clean = np.where(bad[..., None], 0.0, lat)
    byte = nearest(np.clip(np.abs(clean).max(-1) / 6, SCALES[0], SCALES[-1]), SCALES)
    y = np.minimum(np.abs(clean) / SCALES[byte][..., None], 6.0)
    number = nearest(y, LEVELS)
    return number.reshape(-1, 512), np.signbit(lat).reshape(-1, 512), np.where(bad, 255, byte), kv[:, 512:]


def values(kv):
    """What rows [N, 576] read as after the cache, float64 (rope values as they are given)."""
    number, sign, byte, rope = encode(kv)
    scale = np.where(byte == 255, np.nan, SCALES[np.minimum(byte, 247)])
    lat = LEVELS[number] * np.where(sign, -1.0, 1.0)
    return np.concatenate((lat * np.repeat(scale, 16, -1), rope), -1)


def records(kv, rope_bf16_bytes):
    """Rows [N, 576] float64 and their rope values' bf16 bytes uint8 [N, 128] -> records uint8 [N, 416]."""
    number, sign, byte, _ = encode(kv)
    n = kv.shape[0]
    halves = np.zeros((n, 64, 2), np.uint32)                       # word, its 16-bit halves
    num, sg = number.reshape(n, 64, 4, 2).astype(np.uint32), sign.reshape(n, 64, 4, 2).astype(np.uint32)
    for k in range(4):
        halves |= sg[:, :, k] << SIGN[k]
        for bit, at in zip((2, 1, 0), NUMBER[k]):
            halves |= ((num[:, :, k] >> bit) & 1) << at
    words = (halves[..., 0] | halves[..., 1] << 16).astype("<u4").view(np.uint8).reshape(n, 2, 128)
    return np.concatenate((words, byte.astype(np.uint8).reshape(n, 2, 16), rope_bf16_bytes.reshape(n, 2, 64)), -1).reshape(n, 416)


def decode(rec):
    """Records uint8 [N, 416] -> rows float64 [N, 576]."""
    rec = np.ascontiguousarray(rec).reshape(-1, 2, 208)
    h = np.ascontiguousarray(rec[:, :, :128]).view("<u2").reshape(-1, 64, 2).astype(np.int64)
    out = np.zeros((rec.shape[0], 64, 4, 2))
    for k in range(4):
        n = sum(((h >> at) & 1) << bit for bit, at in zip((2, 1, 0), NUMBER[k]))
        out[:, :, k] = LEVELS[n] * np.where((h >> SIGN[k]) & 1, -1.0, 1.0)
    byte = rec[:, :, 128:144].reshape(-1, 32).astype(np.int64)
    scale = np.where(byte == 255, np.nan, SCALES[np.minimum(byte, 247)])
    rope = (np.ascontiguousarray(rec[:, :, 144:]).view("<u2").reshape(-1, 64).astype(np.uint32) << 16).view(np.float32)
    return np.concatenate((out.reshape(-1, 512) * np.repeat(scale, 16, -1), rope.astype(np.float64)), -1)


def attend(q, rec, table, idx, scale, tokens=1):
    """Attention over selected records, float64: q [T, H, 576], rec uint8 [rows, 416], table [B, P], idx [T, K] (-1 = empty)."""
    out = np.zeros((*q.shape[:2], 512))
    for t in range(q.shape[0]):
        pos = idx[t][idx[t] >= 0]
        if len(pos):
            kv = decode(rec[table[t // tokens][pos // PAGE].astype(np.int64) * PAGE + pos % PAGE])
            s = q[t].astype(np.float64) @ kv.T * scale
            p = np.exp(s - s.max(-1, keepdims=True))
            out[t] = (p / p.sum(-1, keepdims=True)) @ kv[:, :512]
    return out


class Pool:
    """Page tables and their rules, one step at a time.  `caches`: arrays [layers, pages * 64, bytes]."""

    def __init__(self, table, ctx, refs, caches=()):
        self.table, self.ctx, self.refs = table.copy(), ctx.copy(), refs.copy()
        self.caches = [c.copy() for c in caches]
        self.status = 0

    def _free(self):
        return [p for p in range(len(self.refs)) if self.refs[p] == 0]

    def _refuse(self, why):
        self.status = self.status or why

    def copy(self, src, dst, tokens=None):
        old = [c.copy() for c in self.caches]
        for i, (s, d) in enumerate(zip(src, dst)):
            if s < 0 or d < 0:
                continue
            if s >= self.caches[0].shape[1] // PAGE or d >= self.caches[0].shape[1] // PAGE:
                self._refuse(2)
                continue
            n = PAGE if tokens is None else min(max(int(tokens[i]), 0), PAGE)
            for c, o in zip(self.caches, old):
                c[:, d * PAGE:d * PAGE + n] = o[:, s * PAGE:s * PAGE + n]

    def extend(self, rows, n_new, max_new):
        B, P = self.table.shape
        slots = np.full((len(rows), max_new), -1, np.int32)
        ok = len(set(map(int, rows))) == len(rows) and all(
            0 <= r < B and 0 <= n <= max_new and self.ctx[r] >= 0 and self.ctx[r] + n <= P * PAGE for r, n in zip(rows, n_new))
        if not ok:
            self._refuse(2)
            return slots
        need = [-(-(int(self.ctx[r]) + int(n)) // PAGE) + -int(self.ctx[r]) // PAGE for r, n in zip(rows, n_new)]
        free = self._free()
        if sum(need) > len(free):
            self._refuse(3)
            return slots
        for i, (r, n) in enumerate(zip(rows, n_new)):
            c, held = int(self.ctx[r]), -(-int(self.ctx[r]) // PAGE)
            for j in range(need[i]):
                self.table[r, held + j] = free.pop(0)
                self.refs[self.table[r, held + j]] = 1
            for t in range(int(n)):
                slots[i, t] = self.table[r, (c + t) // PAGE] * PAGE + (c + t) % PAGE
            self.ctx[r] += n
        return slots

    def fork(self, parents, children):
        B, P = self.table.shape
        kids = list(map(int, children))
        ok = (len(set(kids)) == len(kids) and all(0 <= c < B and self.ctx[c] == 0 for c in kids)
              and all(0 <= p < B and p not in kids and 0 <= self.ctx[p] <= P * PAGE for p in map(int, parents)))
        if not ok:
            return self._refuse(2)
        free = self._free()
        if sum(int(self.ctx[p]) % PAGE != 0 for p in parents) > len(free):
            return self._refuse(3)
        src, dst, tokens = [], [], []
        for p, c in zip(parents, kids):
            n = int(self.ctx[p])
            self.table[c] = -1
            for j in range(n // PAGE):
                self.table[c, j] = self.table[p, j]
                self.refs[self.table[p, j]] += 1
            if n % PAGE:
                new = free.pop(0)
                self.refs[new] = 1
                self.table[c, n // PAGE] = new
                src.append(self.table[p, n // PAGE]), dst.append(new), tokens.append(n % PAGE)
            self.ctx[c] = n
        self.copy(src, dst, tokens)

    def free(self, rows):
        for r in rows:
            if not 0 <= r < len(self.ctx):
                self._refuse(2)
                continue
            for j in range(-(-int(self.ctx[r]) // PAGE)):
                page = self.table[r, j]
                self.table[r, j] = -1
                if 0 <= page < len(self.refs) and self.refs[page] > 0:
                    self.refs[page] -= 1
                else:
                    self._refuse(2)
            self.ctx[r] = 0

    def compact(self):
        used = [p for p in range(len(self.refs)) if self.refs[p] > 0]
        L = len(used)
        high, low = [p for p in reversed(used) if p >= L], [p for p in self._free() if p < L]
        self.copy(high, low)
        to = dict(zip(high, low))
        for h, l in to.items():
            self.refs[l], self.refs[h] = self.refs[h], 0
        for e, page in np.ndenumerate(self.table):
            self.table[e] = to.get(int(page), page)
