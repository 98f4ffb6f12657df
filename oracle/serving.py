"""CPU oracle of the serving operators — TEST INFRASTRUCTURE ONLY (see numerics.py).

The definitions in numpy, 64 bits, one row (or page) after the other.  Attention also returns
what an error bound needs: the sum of |weight * value| and the largest possible rounding error
of a score that was summed in fp32.
"""
from __future__ import annotations

import numpy as np

U32 = 2.0 ** -24      # unit roundoff of fp32
UBF = 2.0 ** -8       # of bf16 (8 significant bits)


def attend(q, k, v, scale, seen):
    """Rows q [R, D] over keys k, v [N, D]; row r sees its first seen[r] keys.

    Returns out [R, D], the same with |v|, lse [R] (-inf without keys), and per row a bound of
    the error that fp32 rounding in a score's sum of D products leaves in it."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    out, mag = np.zeros((len(q), v.shape[1])), np.zeros((len(q), v.shape[1]))
    lse, err = np.full(len(q), -np.inf), np.zeros(len(q))
    for r, n in enumerate(seen):
        if n <= 0:
            continue
        s = (k[:n] @ q[r]) * scale
        top = s.max()
        w = np.exp(s - top)
        z = w.sum()
        out[r], mag[r] = w @ v[:n] / z, w @ np.abs(v[:n]) / z
        lse[r] = top + np.log(z)
        err[r] = (np.abs(k[:n]) @ np.abs(q[r])).max() * scale * (q.shape[1] + 8) * U32
    return out, mag, lse, err


def packed(q, k, v, lens_q, lens_k, scale, causal=True):
    """q [Tq, Hq, D], k / v [Tk, Hkv, D] -> out, magnitude, lse [Tq, Hq], score error."""
    hq, hk = q.shape[1], k.shape[1]
    out, mag = np.zeros(q.shape), np.zeros(q.shape)
    lse, err = np.zeros(q.shape[:2]), np.zeros(q.shape[:2])
    i0 = j0 = 0
    for a, b in zip(lens_q, lens_k):
        seen = [min(b, i + b - a + 1) if causal else b for i in range(a)]
        for h in range(hq):
            kv = h // (hq // hk)
            got = attend(q[i0:i0 + a, h], k[j0:j0 + b, kv], v[j0:j0 + b, kv], scale, seen)
            for dst, x in zip((out, mag, lse, err), got):
                dst[i0:i0 + a, h] = x
        i0, j0 = i0 + a, j0 + b
    return out, mag, lse, err


def paged(q, k_pages, v_pages, table, lens, prefix_len, scale, slots=None):
    """q [B, Hq, D], pages [P, Hkv, page, D] -> out, magnitude, lse, score error.

    A slot that does not exist has no keys; a key whose table entry is no page, or whose row does
    not exist (prefix), is a key and a value of zeros."""
    hq, hk, page = q.shape[1], k_pages.shape[1], k_pages.shape[2]
    slots = range(len(q)) if slots is None else slots
    out, mag = np.zeros(q.shape), np.zeros(q.shape)
    lse, err = np.zeros(q.shape[:2]), np.zeros(q.shape[:2])
    first = list(slots)[0] if len(q) else 0
    for b, s in enumerate(slots):
        n = int(lens[s]) if 0 <= s < len(table) else 0
        if n == 0:
            lse[b] = -np.inf
            continue
        rows = [first if j < prefix_len else s for j in range(n)]
        at = [(table[r][j // page] if 0 <= r < len(table) else -1, j % page)
              for j, r in enumerate(rows)]
        zeros = np.zeros(q.shape[2])
        for h in range(hq):
            kv = h // (hq // hk)
            k, v = (np.array([x[p, kv, o] if 0 <= p < len(x) else zeros
                              for p, o in at]).reshape(n, -1) for x in (k_pages, v_pages))
            o, m, e, x = attend(q[b:b + 1, h], k, v, scale, [n])
            out[b, h], mag[b, h], lse[b, h], err[b, h] = o[0], m[0], e[0], x[0]
    return out, mag, lse, err


def bound(out, mag, err, keys, bf16):
    """How far a kernel may be from `out`.

    With fp32 scores, weights and sums over `keys` keys: each weight is off by the score's error
    (twice: numerator and normaliser), each sum by keys * u of its magnitude; a few u more for
    exp and the division.  In bf16 each weight is rounded once before it meets its value (2^-8
    of the magnitude) and the result once (2^-8 of the result)."""
    fp32 = 4 * (err[..., None] + (keys + 16) * U32) * mag
    return fp32 + (UBF * (mag + np.abs(out)) * 1.01 if bf16 else 2 * U32 * np.abs(out)) + 1e-30


class Pages:
    """The page map of a cache and its pages, changed in place by the same requests."""

    def __init__(self, k, v, table, lens, refs):
        self.k, self.v = np.array(k), np.array(v)
        self.table, self.lens, self.refs = (np.array(x, np.int64) for x in (table, lens, refs))
        self.page = self.k.shape[3]

    def _lowest(self):
        p = int(np.flatnonzero(self.refs == 0)[0])
        self.refs[p] = 1
        return p

    def _release(self, slot):
        for p in self.table[slot][self.table[slot] >= 0]:
            self.refs[p] -= 1
        self.table[slot] = -1
        self.lens[slot] = 0

    def free(self, slots):
        for s in slots:
            self._release(s)

    def fork(self, parents, children):
        for c in children:
            self._release(c)
        for a, c in zip(parents, children):
            full = self.lens[a] // self.page
            self.table[c, :full] = self.table[a, :full]
            for p in self.table[a, :full]:
                self.refs[p] += 1
            self.lens[c] = self.lens[a]
        for a, c in zip(parents, children):
            full, fill = divmod(int(self.lens[a]), self.page)
            if fill:
                src, dst = self.table[a, full], self._lowest()
                self.table[c, full] = dst
                self.k[:, dst, :, :fill] = self.k[:, src, :, :fill]
                self.v[:, dst, :, :fill] = self.v[:, src, :, :fill]

    def reserve(self, slots, lens):
        for s, n in zip(slots, lens):
            for c in range(-(-int(self.lens[s]) // self.page), -(-n // self.page)):
                self.table[s, c] = self._lowest()
            self.lens[s] = n

    def write(self, layer, new_k, new_v, slots, starts, cu):
        for i, s in enumerate(slots):
            for t in range(cu[i], cu[i + 1]):
                pos = starts[i] + t - cu[i]
                p = self.table[s, pos // self.page]
                self.k[layer, p, :, pos % self.page] = new_k[t]
                self.v[layer, p, :, pos % self.page] = new_v[t]

    def compact(self):
        live = [int(p) for p in np.flatnonzero(self.refs > 0)]
        holes = [p for p in range(len(live)) if self.refs[p] == 0]
        for src, dst in zip([p for p in live if p >= len(live)], holes):
            self.k[:, dst], self.v[:, dst] = self.k[:, src], self.v[:, src]
            self.refs[dst], self.refs[src] = self.refs[src], 0
            self.table[self.table == src] = dst

    def copy_pages(self, src, dst):
        for a, b in zip(src, dst):
            self.k[:, b], self.v[:, b] = self.k[:, a], self.v[:, a]


def rope(x, positions, frequencies, factor, layout, inverse=False):
    """x [tokens, heads, D] turned in 64 bits, and |a| + |b| of each element's pair (0: copied)."""
    x = np.asarray(x, np.float64)
    out, mag = x.copy(), np.zeros(x.shape)
    n = 2 * len(frequencies)
    for i, w in enumerate(frequencies):
        a, b = (i, i + n // 2) if layout == "half" else (2 * i, 2 * i + 1)
        angle = np.asarray(positions, np.float64)[:, None] * w
        c, s = factor * np.cos(angle), factor * np.sin(-angle if inverse else angle)
        out[..., a] = x[..., a] * c - x[..., b] * s
        out[..., b] = x[..., b] * c + x[..., a] * s
        mag[..., a] = mag[..., b] = abs(factor) * (np.abs(x[..., a]) + np.abs(x[..., b]))
    return out, mag


BLOCK = 16            # tokens of a page that share a scale
TOP = {"int8": 127.0, "e4m3": 448.0}


def to_code(y, code):
    """y rounded to the nearest code (ties to even), as the number that the code is."""
    y = np.asarray(y, np.float64)
    if code == "int8":
        return np.rint(y)
    step = np.exp2(np.maximum(np.floor(np.log2(np.maximum(np.abs(y), 2.0 ** -60))), -6) - 3)
    return np.rint(y / step) * step


def scale_of(top, code):
    """The least power of two that brings `top` (2^-110 at least) into the codes' range."""
    m, e = np.frexp(np.maximum(top, 2.0 ** -110) / TOP[code])       # 2^e > it >= 2^(e - 1)
    return np.exp2(np.where(m == 0.5, e - 1, e))


class QuantizedPages(Pages):
    """Pages whose k and v hold codes (as numbers), with a scale per block."""

    def __init__(self, k, v, k_scale, v_scale, table, lens, refs, code):
        super().__init__(np.asarray(k, np.float64), np.asarray(v, np.float64), table, lens, refs)
        self.scales = [np.array(x, np.float64) for x in (k_scale, v_scale)]
        self.code = code

    def _moved(self, pairs):
        for a, b in pairs:
            for x in self.scales:
                x[:, b] = x[:, a]

    def fork(self, parents, children):
        super().fork(parents, children)
        self._moved((self.table[a, self.lens[a] // self.page], self.table[c, self.lens[a] // self.page])
                    for a, c in zip(parents, children) if self.lens[a] % self.page)

    def compact(self):
        live = [int(p) for p in np.flatnonzero(self.refs > 0)]
        holes = [p for p in range(len(live)) if self.refs[p] == 0]
        self._moved(zip([p for p in live if p >= len(live)], holes))
        super().compact()

    def copy_pages(self, src, dst):
        super().copy_pages(src, dst)
        self._moved(zip(src, dst))

    def write(self, layer, new_k, new_v, slots, starts, cu):
        for codes, scales, rows in ((self.k, self.scales[0], new_k), (self.v, self.scales[1], new_v)):
            rows = np.asarray(rows, np.float64)
            for i, s in enumerate(slots):
                t, pos = cu[i], int(starts[i])
                while t < cu[i + 1]:
                    r = pos % BLOCK
                    n = min(BLOCK - r, cu[i + 1] - t)
                    p, j, o = self.table[s, pos // self.page], pos % self.page // BLOCK, pos % self.page - r
                    x = rows[t:t + n].transpose(1, 0, 2)
                    finite = np.isfinite(x).all((1, 2))
                    top = np.where(finite, np.abs(np.where(finite[:, None, None], x, 0)).max((1, 2)), 0)
                    scale = np.where(finite, scale_of(top, self.code), np.nan)
                    old = scales[layer, p, :, j]
                    if r:
                        scale = np.where(np.isnan(old), np.nan, np.where(np.abs(old) < scale, scale, old))
                        held = codes[layer, p, :, o:o + r]
                        grown = np.where(np.isnan(scale), 1.0, old / scale)[:, None, None]
                        codes[layer, p, :, o:o + r] = to_code(held * grown, self.code)
                    unit = np.where(np.isnan(scale), np.inf, scale)[:, None, None]
                    y = np.where(np.isfinite(x), x, 0) / unit                  # a NaN block: codes 0
                    codes[layer, p, :, o + r:o + r + n] = to_code(y, self.code)
                    scales[layer, p, :, j] = scale
                    t, pos = t + n, pos + n

    def values(self, layer):
        """(k, v) of a layer as the values that the codes stand for."""
        return tuple(x[layer] * np.repeat(s[layer], BLOCK, -1)[..., None]
                     for x, s in zip((self.k, self.v), self.scales))

    def read(self, layer, slots, starts, cu, out_k, out_v):
        k, v = self.values(layer)
        for i, s in enumerate(slots):
            for t in range(cu[i], cu[i + 1]):
                pos = int(starts[i]) + t - cu[i]
                p = -1
                if 0 <= s < len(self.table) and 0 <= pos < self.lens[s] \
                        and pos // self.page < self.table.shape[1]:
                    p = self.table[s, pos // self.page]
                has = 0 <= p < len(k)
                out_k[t] = k[p, :, pos % self.page] if has else 0
                out_v[t] = v[p, :, pos % self.page] if has else 0
