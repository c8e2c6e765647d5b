"""Paged KV cache in numpy and 64 bits: the page layout of include/e4b_b200.h
(e4b_paged_kv), head prep with the append, and windowed attention with sinks."""
from __future__ import annotations

import numpy as np

F64 = np.float64


def piece_bytes(bits: int, HD: int) -> int:
    return 32 * HD if bits == 16 else 9 * HD


def element_place(bits: int, HD: int, value: bool):
    """For (slot 0..15, dim): byte of its 16-bit word in the piece, and its shift there."""
    s, d = np.arange(16)[:, None], np.arange(HD)[None]
    i, t, z = s // 8 * 2 + s % 2, s // 2 % 4, 0 * (s + d)
    if bits == 16:
        if value:
            return 2 * np.ravel_multi_index((d // 64 + z, i + z, d % 64 // 8 + z, t + z, d % 8 + z), (HD // 64, 4, 8, 4, 8)), z
        return 2 * np.ravel_multi_index((d // 32 + z, s + z, d % 32 + z), (HD // 32, 16, 32)), z
    if value:
        w = np.ravel_multi_index((i + z, d % 32 // 4 + z, t + z, d // 32 + z), (4, 8, 4, HD // 32))
    else:
        nb = min(4, HD // 32)
        w = np.ravel_multi_index((d // 32 // nb + z, s + z, d % 32 // 8 + z, d // 32 % nb + z, d % 8 // 4 + z),
                                 (HD // 32 // nb, 16, 4, nb, 2))
    return HD + 2 * w, 4 * (d % 4) + z


def scale_place(HD: int, value: bool):
    """For (slot, block of 32 dims): byte of its f16 scale in a 4-bit piece."""
    s, b = np.arange(16)[:, None], np.arange(HD // 32)[None]
    if value:
        return 2 * (((s // 2 % 4 * (HD // 32) + b) * 2 + s // 8) * 2 + s % 2)
    return 2 * (s * (HD // 32) + b)


def quantise(x16: np.ndarray):
    """f16 rows [..., HD] -> (codes 0..15, f16 scale per 32 dims): the q4_0 rule with a true division."""
    b = x16.astype(F64).reshape(*x16.shape[:-1], x16.shape[-1] // 32, 32)
    with np.errstate(all="ignore"):
        at = np.abs(b).argmax(-1)
        d = np.take_along_axis(b, at[..., None], -1) / -8.0
        q = np.where(d == 0, 8, np.clip(np.trunc(b / np.where(d == 0, 1.0, d) + 8.5), 0, 15))
        bad = ~np.isfinite(b).all(-1, keepdims=True)
        q = np.where(bad, 8, q).astype(np.int64)
        d16 = np.where(bad, np.nan, d)[..., 0].astype(np.float32).astype(np.float16)
    return q.reshape(x16.shape), d16


def dequantise(q, d16):
    b = (q - 8.0).reshape(*q.shape[:-1], q.shape[-1] // 32, 32) * d16.astype(F64)[..., None]
    return b.reshape(q.shape)


class Pool:
    """One pool (keys or values) as bytes, with element access through the layout's formulas."""

    def __init__(self, bits, page, n_pages, KVH, HD, value, fill=0):
        self.bits, self.page, self.KVH, self.HD, self.value = bits, page, KVH, HD, value
        self.pb = piece_bytes(bits, HD)
        self.raw = np.full(n_pages * KVH * (page // 16) * self.pb, fill, np.uint8)
        self.at, self.shift = element_place(bits, HD, value)
        self.at_d = scale_place(HD, value)

    def _word(self, pageid, head, slot):
        """u16 index of the piece that holds a page's slot."""
        return ((pageid * self.KVH + head) * (self.page // 16) + slot // 16) * self.pb // 2

    def write(self, pageid, slot, rows16):
        """rows16: [KVH][HD] f16 of one token."""
        w = self.raw.view(np.uint16)
        for h in range(self.KVH):
            b, s = self._word(pageid, h, slot), slot % 16
            if self.bits == 16:
                w[b + self.at[s] // 2] = rows16[h].astype(np.float16).view(np.uint16)
                continue
            q, d = quantise(rows16[h].astype(np.float16))
            words = (q.reshape(-1, 4) << np.array([0, 4, 8, 12])).sum(-1)
            w[b + self.at[s][::4] // 2] = words.astype(np.uint16)
            w[b + self.at_d[s] // 2] = d.view(np.uint16)

    def write_all(self, pageids, slots, rows16):
        """As write, for tokens [n]: rows16 [n][KVH][HD]."""
        w, s = self.raw.view(np.uint16), slots % 16
        b = self._word(pageids[:, None], np.arange(self.KVH)[None], slots[:, None])[..., None]
        if self.bits == 16:
            w[b + self.at[s][:, None] // 2] = rows16.astype(np.float16).view(np.uint16)
            return
        q, d = quantise(rows16.astype(np.float16))
        words = (q.reshape(*q.shape[:-1], q.shape[-1] // 4, 4) << np.array([0, 4, 8, 12])).sum(-1)
        w[b + self.at[s][:, None, ::4] // 2] = words.astype(np.uint16)
        w[b + self.at_d[s][:, None] // 2] = d.view(np.uint16)

    def read_all(self, pageids, slots):
        """As read, for tokens [n]: [n][KVH][HD] in 64 bits."""
        w, s = self.raw.view(np.uint16), slots % 16
        b = self._word(pageids[:, None], np.arange(self.KVH)[None], slots[:, None])[..., None]
        x = w[b + self.at[s][:, None] // 2]
        if self.bits == 16:
            return x.view(np.float16).astype(F64)
        return dequantise(((x >> self.shift[s][:, None]) & 15).astype(F64), w[b + self.at_d[s][:, None] // 2].view(np.float16))

    def read(self, pageid, slot):
        """[KVH][HD] in 64 bits."""
        w = self.raw.view(np.uint16)
        out = np.zeros((self.KVH, self.HD))
        for h in range(self.KVH):
            b, s = self._word(pageid, h, slot), slot % 16
            x = w[b + self.at[s] // 2]
            if self.bits == 16:
                out[h] = x.view(np.float16).astype(F64)
            else:
                out[h] = dequantise(((x >> self.shift[s]) & 15).astype(F64), w[b + self.at_d[s] // 2].view(np.float16))
        return out


def headprep(x, pos, qw, kw, QH, KVH, HD, angles, theta, eps, norm, keqv):
    """Rows x [n][heads*HD] at positions pos -> (q, k, v) in 64 bits, before any rounding."""
    x = x.astype(F64).reshape(len(pos), -1, HD)
    q, k = x[:, :QH], x[:, QH:QH + KVH]
    v = k if keqv else x[:, QH + KVH:QH + 2 * KVH]
    if norm:
        q, k, v = (t / np.sqrt((t * t).mean(-1, keepdims=True) + F64(np.float32(eps))) for t in (q, k, v))
        k = k * kw.astype(F64)
        q = q * qw.astype(F64) if QH else q
    a = np.asarray(pos, F64)[:, None, None] * F64(np.float32(theta)) ** (-2.0 * np.arange(angles) / HD)
    h = HD // 2

    def turn(t):
        t = t.copy()
        x0, x1 = t[..., :angles].copy(), t[..., h:h + angles].copy()
        t[..., :angles] = x0 * np.cos(a) - x1 * np.sin(a)
        t[..., h:h + angles] = x0 * np.sin(a) + x1 * np.cos(a)
        return t

    return turn(q), turn(k), v


def visible(n_slots, p, window, sinks):
    t = np.arange(n_slots)
    return (t <= p) & ((window == 0) | (t > p - window) | (t < sinks))


def attention(q, p, k, v, window, sinks, scale, usable=None):
    """One row: q [QH][HD] at position p over k, v [slots][KVH][HD] -> (o [QH][HD], lse [QH])."""
    QH, HD = q.shape
    KVH = k.shape[1]
    see = visible(len(k), p, window, sinks)
    if usable is not None:
        see &= usable
    o, lse = np.zeros((QH, HD)), np.full(QH, -np.inf)
    if see.any():
        for h in range(QH):
            s = scale * (k[see, h // (QH // KVH)] @ q[h].astype(F64))
            m = s.max()
            e = np.exp(s - m)
            lse[h] = m + np.log(e.sum())
            o[h] = e @ v[see, h // (QH // KVH)] / e.sum()
    return o, lse
