"""The paged KV cache in 4 bits restated plainly, in numpy and 64 bits: where an element lies in a
page, how a block is quantized, what the page calls do to tables, lengths, reference counts and
pages, and attention over what a sequence holds. The tests compare the library with it."""
from __future__ import annotations

import numpy as np


def place(hd, pos, dim, value):
    """(byte of the code, shift of its nibble, byte of its scale) in the 36 * hd bytes of the tile of
    32 positions of one head."""
    if value:
        e = pos // 16 * 4 + pos % 4
        g = pos % 16 // 4
        dword = ((dim // 64 * 4 + g) * 16 + dim % 16) * 4 + dim // 16 % 4
        byte, scale = 16 * hd + 4 * dword, 34 * hd + 2 * ((dim // 32 * 4 + g) * 8 + e)
    else:
        w = min(4, hd // 32)
        g, inner = dim // (hd // 4), dim % (hd // 4)
        e, j = inner % 8, inner // 8
        dword = (((pos // 16 * (hd // 32 // w) + j // w) * 4 + g) * 16 + pos % 16) * w + j % w
        byte, scale = 4 * dword, 32 * hd + 2 * ((dim // 32 * 16 + pos % 16) * 2 + pos // 16)
    nibble = e // 2 + 4 * (e % 2)
    return byte + nibble // 2, nibble % 2 * 4, scale


def places(hd, value):
    """place() over [32][hd]: three integer arrays."""
    out = np.empty((3, 32, hd), np.int64)
    for p in range(32):
        for d in range(hd):
            out[:, p, d] = place(hd, p, d, value)
    return out


def round_bits(x, bits):
    """x rounded to `bits` significant bits, half to even (float64)."""
    m, e = np.frexp(x)
    return np.ldexp(np.round(np.ldexp(m, bits)), e - bits)


def quantize(x):
    """x [..., hd] float32 -> (codes, scales): the definition in 64 bits. Finite rows."""
    b = x.astype(np.float64).reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    mx, mn = b.max(-1), b.min(-1)
    a = np.minimum(round_bits(np.maximum(mx, -mn) / 8, 8), 8160.0)
    a = np.where(a < 2.0 ** -14, np.round(a * 2.0 ** 24) * 2.0 ** -24, a)  # fp16's grid
    d = np.where(-mn >= mx, a, -a)
    dd = np.where(d == 0, 1.0, d)[..., None]
    c = np.where((d == 0)[..., None], 8, np.clip(np.round(b / dd) + 8, 0, 15)).astype(np.int64)
    return c.reshape(x.shape), d


def stored(k, v):
    """What the rows k and v [..., hd] float32 of a head read back as (float64)."""
    bad = ~(np.isfinite(k).all(-1) & np.isfinite(v).all(-1))
    out = []
    for x, fill in ((k, np.nan), (v, 0.0)):
        c, d = quantize(np.where(bad[..., None], np.float32(0), x))
        y = ((c - 8).reshape(*d.shape, 32) * d[..., None]).reshape(x.shape)
        out.append(np.where(bad[..., None], fill, y))
    return out


class Cache:
    """Tables, lengths, counts and the pages' values, one call after the other."""

    def __init__(self, n_layers, n_pages, max_seqs, max_pages, page_size, n_kv, hd):
        self.page = page_size
        self.table = np.full((max_seqs, max_pages), -1, np.int64)
        self.lens = np.zeros(max_seqs, np.int64)
        self.refs = np.zeros(n_pages, np.int64)
        self.kv = np.zeros((2, n_layers, n_pages, page_size, n_kv, hd))

    def _pages(self, n):
        return -(-n // self.page)

    def extend(self, slots, counts):
        seen, plan = set(), []
        refs = self.refs.copy()
        for s, c in zip(slots, counts):
            if not 0 <= s < len(self.lens) or s in seen or c < 0:
                return -1
            seen.add(s)
            n = int(self.lens[s])
            if self._pages(n + c) > self.table.shape[1]:
                return -1
            copy = False
            if c > 0 and n % self.page:
                p = self.table[s, self._pages(n) - 1]
                if not 0 <= p < len(refs):
                    return -1
                copy = refs[p] > 1
                if copy:
                    refs[p] -= 1
            plan.append((s, c, copy))
        need = sum(copy + self._pages(int(self.lens[s]) + c) - self._pages(int(self.lens[s])) for s, c, copy in plan)
        free = [int(i) for i in np.flatnonzero(self.refs == 0)]
        if need > len(free):
            return need - len(free)
        self.refs = refs
        at = 0
        for s, c, copy in plan:
            n = int(self.lens[s])
            if copy:
                last = self._pages(n) - 1
                self.kv[:, :, free[at]] = self.kv[:, :, self.table[s, last]]
                self.table[s, last] = free[at]
                self.refs[free[at]] = 1
                at += 1
            for j in range(self._pages(n), self._pages(n + c)):
                self.table[s, j] = free[at]
                self.refs[free[at]] = 1
                at += 1
            self.lens[s] = n + c
        return 0

    def _release(self, s, first=0):
        for p in self.table[s, first:]:
            if 0 <= p < len(self.refs):
                self.refs[p] -= 1
        self.table[s, first:] = -1

    def fork(self, src, dst):
        rows, lens, named, todo = {}, {}, set(), []
        for s, d in zip(src, dst):
            if d in named or not 0 <= d < len(self.lens):
                continue
            named.add(d)
            if 0 <= s < len(self.lens):
                todo.append(d)
                rows[d], lens[d] = self.table[s].copy(), self.lens[s]
        for d in todo:
            for p in rows[d]:
                if 0 <= p < len(self.refs):
                    self.refs[p] += 1
        for d in todo:
            self._release(d)
            self.table[d], self.lens[d] = rows[d], lens[d]

    def truncate(self, slots, new_lens=None):
        named = set()
        for i, s in enumerate(slots):
            if s in named or not 0 <= s < len(self.lens):
                continue
            named.add(s)
            n = min(int(self.lens[s]), max(0, int(new_lens[i]) if new_lens is not None else 0))
            self._release(s, self._pages(n))
            self.lens[s] = n

    def compact(self):
        live = self.refs > 0
        n = int(live.sum())
        moved = [i for i in range(n, len(live)) if live[i]]
        holes = [i for i in range(n) if not live[i]]
        for s, d in zip(moved, holes):
            self.kv[:, :, d] = self.kv[:, :, s]
            self.refs[d], self.refs[s] = self.refs[s], 0
            self.table[self.table == s] = d
        return n

    def positions(self, s, r):
        """Position of each of the last r rows of slot s."""
        return int(self.lens[s]) - r + np.arange(r)

    def store(self, layer, s, k, v):
        """k, v [r, n_kv, hd] float32: the last r tokens of slot s."""
        kk, vv = stored(k, v)
        for t, p in enumerate(self.positions(s, len(k))):
            if p < 0:
                continue
            page = self.table[s, p // self.page]
            if 0 <= page < len(self.refs):
                self.kv[0, layer, page, p % self.page] = kk[t]
                self.kv[1, layer, page, p % self.page] = vv[t]

    def rows(self, layer, s, n):
        """(keys, values [n, n_kv, hd], whether the position has a page) of slot s."""
        p = np.arange(n)
        page = self.table[s, p // self.page]
        ok = (page >= 0) & (page < len(self.refs))
        page = np.where(ok, page, 0)
        kv = self.kv[:, layer, page, p % self.page]
        return np.where(ok[:, None, None], kv[0], 0.0), np.where(ok[:, None, None], kv[1], 0.0), ok


def attention(q, k, v, ok, first):
    """q [r, n_head, hd] over k, v [n, n_kv, hd] in 64 bits; row t sees positions <= first + t that
    are ok. Returns the outputs, and per output the bounds the tolerance is made of: the largest
    sum |q_i k_i| / sqrt(hd) of the row's positions, sum p |v| and sum |v|."""
    r, n_head, hd = q.shape
    n, n_kv = k.shape[:2]
    g = n_head // n_kv
    q = q.astype(np.float64).reshape(r, n_kv, g, hd)
    out, size, mass, total = (np.zeros((r, n_kv, g, hd)) for _ in range(4))
    for h in range(n_kv):
        s = np.einsum("rgd,nd->rgn", q[:, h], k[:, h]) / np.sqrt(hd)
        a = np.einsum("rgd,nd->rgn", np.abs(q[:, h]), np.abs(k[:, h])) / np.sqrt(hd)
        size_v = np.abs(v[:, h])
        for t in range(r):
            seen = ok & (np.arange(n) <= first + t)
            if not seen.any():
                continue
            x = s[t][:, seen]
            p = np.exp(x - x.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            out[t, h] = p @ v[seen, h]
            mass[t, h] = p @ size_v[seen]
            total[t, h] = size_v[seen].sum(0)
            size[t, h] = a[t][:, seen].max(-1, keepdims=True)
    return [x.reshape(r, n_head, hd) for x in (out, size, mass, total)]


def attention_bound(hd, n, size, mass, total):
    """How far the kernel may be from the exact output. The keys and values enter exactly. A query
    element as two fp16 parts is off by at most 2^-20 of itself, the fp32 accumulation of hd products by
    (hd + 8) 2^-24 of their magnitudes, the scaling to log2 units, the subtraction of the maximum and the
    exponential by 2^-21 of the score's size and 2^-22; so a weight is off by at most d below, relatively, and the
    quotient of two sums of weights by 2 d. A weight as two fp16 parts, the largest between 2^11 and 2^15,
    adds 2^-20 of itself, or 2^-24 below fp16's normal numbers, 2^-35 of the largest: that times sum |v| in all,
    as the weights' sum is at least the largest (an output whose values lie under small weights only
    keeps an absolute accuracy). The running sums of a wave add one rounding per step:
    n / 16 of the denominator, n / 128 of the outputs, and the joins some 64."""
    d = size * (2.0 ** -20 + (hd + 8) * 2.0 ** -24 + 2.0 ** -21) + 2.0 ** -21
    return mass * (2.2 * d + 2.0 ** -20 + (n / 16 + n / 128 + 64) * 2.0 ** -24) + 2.0 ** -35 * total


def attention_rms_bound():
    """And how far in the root mean square over all outputs, relative to theirs: every error above is a
    rounding, of either sign (the parts' truncations follow the signs of the elements they truncate), so
    over hd products and many outputs the largest of them, 2^-20 of a score of unit spread and of a weight,
    counts about once: 4 * 2^-20 covers both, the accumulations and the values' spread. (A loss of bits
    common to all terms, as of subnormal operands that are not normalised, is 2^-16 here.)"""
    return 2.0 ** -18
