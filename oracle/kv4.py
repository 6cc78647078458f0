"""Paged 4-bit KV cache, restated in numpy: the bytes of a block, the bookkeeping of a pool and attention in 64 bits."""
from __future__ import annotations

import numpy as np


def quantise(x):
    """x fp32 [..., D] -> codes int [..., D] and scales fp16 [..., D / 32]: scale = fp16(min(absmax * fp32(1/7), 65504)), code =
    clip(rint(x / scale), +-7)."""
    g = np.ascontiguousarray(x, dtype=np.float32).reshape(*x.shape[:-1], -1, 32)
    s = np.minimum(np.abs(g).max(-1) * (np.float32(1) / np.float32(7)), np.float32(65504)).astype(np.float16)
    s32 = s.astype(np.float32)[..., None]
    c = np.clip(np.rint(g / np.where(s32 > 0, s32, np.float32(1))), -7, 7)
    return np.where(s32 > 0, c, 0).astype(np.int32).reshape(x.shape), s


def held(x):
    """What the cache holds of rows x, in 64 bits."""
    codes, scales = quantise(x)
    return codes * np.repeat(scales.astype(np.float64), 32, axis=-1)


def code_place(r, d, values: bool):
    """(byte within the codes of a block, nibble) of position r, dimension d."""
    G, i, e = d // 32, d % 32 // 16, d % 16
    if not values:
        return G * 256 + ((r % 8) * 4 + e % 8 // 2) * 8 + 4 * i + r // 8 + 2 * (e % 2), e // 8
    return G * 256 + ((e % 8) * 4 + r % 8 // 2) * 8 + 4 * i + r // 8 + 2 * (r % 2), e // 8


def block_bytes(k, v):
    """The 576 * D / 32 bytes of a block of 16 rows k, v fp32 [16, D]."""
    D = k.shape[1]
    NG, out = D // 32, []
    for values, x in ((False, k), (True, v)):
        codes, scales = quantise(x)
        b = np.zeros(8 * D, np.uint8)
        s = np.zeros(D // 2, np.float16)
        for r in range(16):
            for d in range(D):
                byte, high = code_place(r, d, values)
                b[byte] |= (codes[r, d] + 8) << (4 * high)
            for G in range(NG):
                s[G * 16 + r % 8 // 2 * 4 + r // 8 * 2 + r % 2 if values else r * NG + G] = scales[r, G]
        out += [b, s.view(np.uint8)]
    return np.concatenate(out)


def attention(q, K, V, first: int):
    """q [n, Hq, D], K and V [len, Hkv, D] in 64 bits; row i sees positions 0 .. first + i.  -> (o, sum_p p |v|, the largest
    sum_d |q_d k_d| / sqrt(D) over the positions each row sees) with o [n, Hq, D]."""
    n, Hq, D = q.shape
    rep = Hq // K.shape[1]
    q, K, V = (x.astype(np.float64) for x in (q, K, V))
    o, mag, size = np.zeros_like(q), np.zeros_like(q), np.zeros((n, Hq, 1))
    for i in range(n):
        for h in range(Hq):
            k, v = K[:first + i + 1, h // rep], V[:first + i + 1, h // rep]
            s = k @ q[i, h] / np.sqrt(D)
            p = np.exp(s - s.max())
            p /= p.sum()
            o[i, h], mag[i, h] = p @ v, p @ np.abs(v)
            size[i, h] = (np.abs(k) @ np.abs(q[i, h])).max() / np.sqrt(D)
    return o, mag, size


class Pool:
    """Page tables, lengths and reference counts; `data[page]` names what a page holds (any value per position)."""

    def __init__(self, n_pages, max_seqs, max_pages, page):
        self.page, self.max_pages = page, max_pages
        self.tables = np.full((max_seqs, max_pages), -1, np.int32)
        self.lens, self.refs = np.zeros(max_seqs, np.int32), np.zeros(n_pages, np.int32)

    def _count(self, n):
        return -(-n // self.page)

    def extend(self, slots, rows):
        """-> pos, [(from, to)] page copies.  Everything is decided from the state before the call."""
        refs, free = self.refs.copy(), [i for i, r in enumerate(self.refs) if r == 0]
        pos, copies, taken, seen = [], [], 0, set()
        for s, n in zip(slots, rows):
            if s in seen or not 0 <= s < len(self.lens) or n < 0 or self.lens[s] + n > self.page * self.max_pages:
                pos.append(-1)
                continue
            seen.add(s)
            len_ = int(self.lens[s])
            had, has = self._count(len_), self._count(len_ + n)
            cow = int(n > 0 and len_ % self.page != 0 and refs[self.tables[s, had - 1]] > 1)
            need, at = has - had + cow, taken
            if need > len(free) - taken:                 # not enough left; the ones behind it are served all the same
                pos.append(-1)
                continue
            taken += need
            new = free[at:at + need]
            if cow:
                old = int(self.tables[s, had - 1])
                copies.append((old, new[0]))
                self.refs[old] -= 1
            self.tables[s, had - cow:has] = new
            self.refs[new] = 1
            self.lens[s] = len_ + n
            pos.append(len_)
        return pos, copies

    def fork(self, src, dst):
        old = [(self.tables[s].copy(), int(self.lens[s])) for s in src]
        last = {d: i for i, d in enumerate(dst)}
        for d, i in last.items():
            row, n = old[i]
            self.refs[row[:self._count(n)]] += 1
        for d, i in last.items():
            self.refs[self.tables[d, :self._count(int(self.lens[d]))]] -= 1
            self.tables[d], self.lens[d] = old[i]

    def free(self, slots):
        for s in slots:
            self.refs[self.tables[s, :self._count(int(self.lens[s]))]] -= 1
            self.tables[s], self.lens[s] = -1, 0

    def compact(self, n_pages):
        """-> the other pool, and the old numbers of its pages."""
        live = np.flatnonzero(self.refs > 0)
        to = Pool(n_pages, len(self.lens), self.max_pages, self.page)
        new = np.full(len(self.refs) + 1, -1, np.int32)
        new[live] = np.arange(len(live))
        to.tables, to.lens = new[self.tables], self.lens.copy()
        to.refs[:len(live)] = self.refs[live]
        return to, live
