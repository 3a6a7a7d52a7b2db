"""What stands between the q|k|v projection and the output projection, in numpy (test infrastructure only): the heads' rules in fp32, an operation and
its rounding after the other, and in 64 bits; the paged cache's bytes; attention in 64 bits."""
from __future__ import annotations

import numpy as np

from oracle import qwmx

PLUS_ONE, PAIRS, FWHT_QK, FWHT_V = 1, 2, 4, 8


def table(positions: int, rope: int, base: float = 10000.0) -> np.ndarray:
    angle = np.arange(positions)[:, None] * base ** (-np.arange(0, rope, 2) / rope)
    return np.concatenate([np.cos(angle), np.sin(angle)], 1).astype(np.float32)


def _halve(t):
    while t.shape[-1] > 1:
        t = t[..., : t.shape[-1] // 2] + t[..., t.shape[-1] // 2:]
    return t[..., 0]


def fwht32(x):
    y = x.reshape(-1, 32)
    for h in (1, 2, 4, 8, 16):
        y = y.reshape(-1, 16 // h, 2, h)
        y = np.stack([y[:, :, 0] + y[:, :, 1], y[:, :, 0] - y[:, :, 1]], 2).reshape(-1, 32)
    return (y * y.dtype.type(np.float32(1.0 / np.sqrt(32.0)) if y.dtype == np.float32 else 1.0 / np.sqrt(32.0))).reshape(x.shape)


def heads(x, gamma=None, plus_one=False, eps=1e-6, cos_sin=None, position=None, pairs=False, fwht=False, dtype=np.float32):
    """x [rows, heads, d] -> the same shape in `dtype` (np.float32: the door's own operations and order; np.float64: the definition)."""
    t = np.dtype(dtype).type
    x = x.astype(dtype)
    d = x.shape[-1]
    with np.errstate(all="ignore"):
        if gamma is not None:
            s = _halve((x * x).reshape(*x.shape[:-1], d // 8, 8))
            room = 1 << (d // 8 - 1).bit_length()
            s = _halve(np.concatenate([s, np.zeros((*s.shape[:-1], room - d // 8), dtype)], -1))
            r = t(1.0) / np.sqrt(s * (t(1.0) / t(d)) + t(np.float32(eps)))
            g = gamma.astype(dtype)
            x = (x * r[..., None]) * (t(1.0) + g if plus_one else g)
        if cos_sin is not None:
            n = cos_sin.shape[1]
            row = cos_sin[np.clip(position, 0, len(cos_sin) - 1)].astype(dtype)[:, None]
            c, s = row[..., : n // 2], row[..., n // 2:]
            y = x.copy()
            a, b = (x[..., 0:n:2], x[..., 1:n:2]) if pairs else (x[..., : n // 2], x[..., n // 2:n])
            u, v = a * c - b * s, b * c + a * s
            if pairs:
                y[..., 0:n:2], y[..., 1:n:2] = u, v
            else:
                y[..., : n // 2], y[..., n // 2:n] = u, v
            x = y
        if fwht:
            x = fwht32(x)
    return x


class Cache:
    """Pages as the doors keep them."""

    def __init__(self, pages, page, heads, d, fill=0):
        self.page, self.heads, self.d = page, heads, d
        self.bytes = np.full((pages, heads, page * d * 34 // 32), fill, np.uint8)

    def planes(self):
        """Views: keys' codes [pages, heads, page, d / 2], their scales, values' codes [pages, heads, page / 8, d / 8, 8, 4], their scales [.., page / 8, d / 32, 8]."""
        p, d = self.page, self.d
        a, b = p * d // 2, p * d // 32
        n, h, _ = self.bytes.shape
        kc, ks, vc, vs = (self.bytes[:, :, i:j] for i, j in ((0, a), (a, a + b), (a + b, 2 * a + b), (2 * a + b, 2 * a + 2 * b)))
        # reshaping a slice of the last axis keeps it a view
        return (_split(kc, (p, d // 2)), _split(ks, (p, d // 32)), _split(vc, (p // 8, d // 8, 8, 4)), _split(vs, (p // 8, d // 32, 8)))

    def put(self, slots, k, v):
        """k, v [rows, heads, d] of any float type: quantised and written at the slots (negative: skipped)."""
        kc, ks, vc, vs = self.planes()
        rows, heads, d = k.shape
        (c, s), (e, f) = (qwmx.quantise(x.reshape(rows * heads, d)) for x in (k, v))
        c, e = c.reshape(rows, heads, d // 2), e.reshape(rows, heads, d // 2)
        s, f = s.reshape(rows, heads, d // 32), f.reshape(rows, heads, d // 32)
        for r in range(rows):
            if 0 <= slots[r] < len(self.bytes) * self.page:
                p, t = divmod(int(slots[r]), self.page)
                kc[p, :, t], ks[p, :, t] = c[r], s[r]
                vc[p, :, t // 8, :, t % 8], vs[p, :, t // 8, :, t % 8] = e[r].reshape(heads, d // 8, 4), f[r]

    def tokens(self, pages, length):
        """Keys and values f64 [heads, length, d] of the sequence with these pages; scale bytes over 252 read as NaN."""
        kc, ks, vc, vs = (x[np.asarray(pages)[: -(-length // self.page)]] for x in self.planes())
        n, h, p, d = len(kc), self.heads, self.page, self.d
        vc = vc.transpose(0, 1, 2, 4, 3, 5).reshape(n, h, p, d // 2)
        vs = vs.transpose(0, 1, 2, 4, 3).reshape(n, h, p, d // 32)
        return tuple(qwmx.values(c.reshape(-1, d // 2), np.where(s > 252, 255, s).reshape(-1, d // 32)).reshape(n, h, p, d).transpose(1, 0, 2, 3).reshape(h, n * p, d)[:, :length]
                     for c, s in ((kc, ks), (vc, vs)))


def _split(x, shape):
    strides, step = [], x.strides[-1]
    for n in reversed(shape):
        strides.insert(0, step)
        step *= n
    return np.lib.stride_tricks.as_strided(x, x.shape[:-1] + tuple(shape), x.strides[:-1] + tuple(strides))


def attention(q, k, v, scale, window=0):
    """q f64 [n, q_heads, d] of a sequence's last rows, k, v f64 [heads, length, d] -> out [n, q_heads, d], lse [n, q_heads], and sum p |v| (what bounds the
    rounding of the weights).  A token that a row does not see does not reach it, a NaN neither."""
    n, heads, d = q.shape
    shared, length = heads // k.shape[0], k.shape[1]
    out, lse, size = np.zeros(q.shape), np.full((n, heads), -np.inf), np.zeros(q.shape)
    with np.errstate(all="ignore"):
        for i in range(n):
            pos = length - n + i
            lo = max(0, pos - window + 1) if window else 0
            if pos < lo:
                continue
            for h in range(heads):
                kk, vv = k[h // shared, lo:pos + 1], v[h // shared, lo:pos + 1]
                s = (kk @ q[i, h]) * scale
                m = np.nanmax(s) if not np.isnan(s).all() else np.nan
                p = np.exp(s - m)
                lse[i, h] = m + np.log(p.sum())
                p = p / p.sum()
                out[i, h] = p @ vv
                size[i, h] = p @ np.abs(vv)
    return out, lse, size
