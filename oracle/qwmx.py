"""MXFP4 and the logits' rules in numpy: the definitions, value by value, in 64 bits (test infrastructure only)."""
from __future__ import annotations

import numpy as np

from oracle import qworacle as qo

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
BORDERS = 0.5 * (GRID[1:] + GRID[:-1])
SIGNED = np.concatenate([GRID, -GRID])


def quantise(x: np.ndarray):
    """x [rows, k] of any float type -> (codes u8 [rows, k / 2], scales u8 [rows, k / 32])."""
    rows, k = x.shape
    v = x.astype(np.float64).reshape(rows, k // 32, 32)
    broken = ~np.isfinite(v).all(axis=2)
    a = np.abs(np.where(np.isfinite(v), v, 0.0))
    _, e = np.frexp(a.max(axis=2))                       # a = m 2^e, 1/2 <= m < 1: floor(log2 a) = e - 1
    e = np.where(a.max(axis=2) > 0, np.maximum(e - 3, -127), -127)
    t = a / np.exp2(e.astype(np.float64))[:, :, None]
    low, high = np.searchsorted(BORDERS, t, side="left"), np.searchsorted(BORDERS, t, side="right")
    mag = np.where(low == high, low, np.where(low % 2 == 0, low, high))   # on a border: the even code
    code = mag.astype(np.uint8) | (np.signbit(v).astype(np.uint8) << 3)
    code = np.where(broken[:, :, None], 0, code).astype(np.uint8).reshape(rows, k // 2, 2)
    scales = np.where(broken, 255, e + 127).astype(np.uint8)
    return code[:, :, 0] | (code[:, :, 1] << 4), scales


def values(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """f64 [rows, k]."""
    rows, half = codes.shape
    v = np.empty((rows, half * 2))
    v[:, 0::2], v[:, 1::2] = SIGNED[codes & 15], SIGNED[codes >> 4]
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127.0))
    return v * np.repeat(s, 32, axis=1)


def logits_f32(l, hist=None, prompt=None, total=None, rep=None, pres=None, freq=None, bias=None, allowed=None, allowed_row=None):
    """The rules in fp32, one rounding an operation (what the door promises); bias: a list of (token, value) lists, allowed: bool [masks, n].
    Returns (fp32 results [rows, n], tokens)."""
    l = l.astype(np.float32).copy()
    rows, n = l.shape
    one = np.float32(1.0)
    tokens = np.empty(rows, np.int32)
    with np.errstate(all="ignore"):
        for r in range(rows):
            if hist is not None:
                t = hist[r, :max(0, min(int(total[r]), hist.shape[1]))]
                p = int(prompt[r]) if prompt is not None else 0
                inside = (t >= 0) & (t < n)
                seen = np.bincount(t[inside], minlength=n) > 0
                answer = inside & (np.arange(len(t)) >= p)
                count = np.bincount(t[answer], minlength=n)
                rr = one if rep is None else np.float32(rep[r])
                l[r] = np.where(seen, np.where(l[r] > 0, l[r] / rr, l[r] * rr), l[r])
                ff, pp = np.float32(0 if freq is None else freq[r]), np.float32(0 if pres is None else pres[r])
                l[r] = np.where(count > 0, (l[r] - ff * count.astype(np.float32)) - pp, l[r])
            if bias is not None:
                for tok, val in dict(bias[r]).items():     # dict(): the later entry of a token
                    if 0 <= tok < n:
                        l[r, tok] = l[r, tok] + np.float32(val)
            if allowed is not None:
                at = r if allowed_row is None else int(allowed_row[r])
                if 0 <= at < len(allowed):
                    l[r] = np.where(allowed[at], l[r], -np.inf)
            tokens[r] = qo.head_argmax(l[r])[0] if (l[r] > -np.inf).any() else -1   # the key rule: +0 is above -0
    return l, tokens
