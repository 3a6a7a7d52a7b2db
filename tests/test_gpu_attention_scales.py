"""qwhip_kv_attention_mxfp4 where blocks outside of the half types' range decide the result, with a bound for each output of its own.

Bound of element i of a row and head, all sums over the tokens t that the row sees: half a step of the type of |o|; 2^-11 sum p |v| for the weights' rounding to f16, fp32's sum of n products
n 2^-24 of the same; sum p e_t (|v| + |o|) for the scores, e_t = (D + 8) 2^-24 scale sum |q k_t| + 2^-20; 2^-37 sum |v| where weights are subnormal in f16.
Each test shows on its own data that reading the blocks in question as zero would be far out of these bounds."""
import numpy as np
import pytest

from qwegn_amd import qwhip
from tests.test_gpu_attention import HALF_STEP, Case
from tests.test_gpu_attention_tiles import Tiles
from tests.test_gpu_heads import decode, encode

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return qwhip.Device(0)


def outputs(q, k, v, scale, t):
    """q f64 [n, heads, d] of the last rows, k, v f64 [length, d] of their one key head -> out, its bound, the logarithm of the sum, its bound."""
    n, heads, d = q.shape
    length = len(k)
    seen = np.arange(length)[None] <= np.arange(length - n, length)[:, None]
    res = [np.empty(q.shape), np.empty(q.shape), np.empty((n, heads)), np.empty((n, heads))]
    for h in range(heads):
        s = np.where(seen, q[:, h] @ k.T * scale, -np.inf)
        e = (d + 8) * 2.0 ** -24 * (np.abs(q[:, h]) @ np.abs(k).T) * scale + 2.0 ** -20
        m = s.max(1, keepdims=True)
        p = np.exp(s - m)
        total = p.sum(1, keepdims=True)
        p /= total
        o, size, moved = p @ v, p @ np.abs(v), p * e
        res[0][:, h] = o
        res[1][:, h] = HALF_STEP[t] * np.abs(o) + (2.0 ** -11 * 1.01 + length * 2.0 ** -24) * size + moved @ np.abs(v) + moved.sum(1, keepdims=True) * np.abs(o) + \
            2.0 ** -37 * (seen @ np.abs(v)) + (2.0 ** -25 if t == "f16" else 0.0)
        res[2][:, h] = (m + np.log(total))[:, 0]
        res[3][:, h] = moved.sum(1) + 2.0 ** -22 * (np.abs(res[2][:, h]) + np.log(length + 2.0))
    return res


# which plane, its scale bytes, the queries' magnitude
KINDS = {("small values", "f16"): ("v", 110, 113, 1.0), ("small values", "bf16"): ("v", 100, 113, 1.0), ("smallest values", "bf16"): ("v", 30, 60, 1.0), ("large values", "bf16"): ("v", 141, 220, 1.0),
         ("small keys", "f16"): ("k", 100, 113, 2.0 ** 10), ("small keys", "bf16"): ("k", 60, 113, 2.0 ** 30), ("large keys", "f16"): ("k", 141, 150, 2.0 ** -6),
         ("large keys", "bf16"): ("k", 141, 180, 2.0 ** -30)}


@pytest.mark.parametrize("cls,d,page,rows,lengths", [(Case, 64, 16, [1, 20, 5], [200, 333, 64]), (Case, 128, 64, [1, 20, 5], [200, 333, 64]), (Case, 256, 16, [1, 20, 5], [200, 333, 64]),
                                                      (Tiles, 64, 16, [80, 5, 1], [180, 333, 64]), (Tiles, 128, 64, [80, 5, 1], [180, 333, 64])])
@pytest.mark.parametrize("kind", sorted(KINDS), ids="-".join)
def test_blocks_that_decide(dev, cls, d, page, rows, lengths, kind):
    """All blocks of a head's keys or values out of range, the other head ordinary."""
    t, (plane, low, high, size) = kind[1], KINDS[kind]
    rng = np.random.default_rng(d)
    c = cls(dev, 3, d, 2, 4, page, rows, lengths, t)
    kc, ks, vc, vs = c.cache.planes()
    target, codes = (ks, kc) if plane == "k" else (vs, vc)
    target[:, 0] = rng.integers(low, high + 1, target[:, 0].shape)
    q = decode(c.q, t).astype(np.float64)
    if plane == "k":
        k, _ = c.cache.tokens(c.table[0], lengths[0])
        q[:, :4] *= size
        c.q = encode(q, t)
        q = decode(c.q, t).astype(np.float64)
        c.scale = np.float32(3.0 / (q[:, :4] @ k[0].T).std())                             # scores that differ by some
        q[:, 4:] *= 1.0 / float(c.scale)
        c.q = encode(np.clip(q, -3e4, 3e4) if t == "f16" else q, t)
        q = decode(c.q, t).astype(np.float64)
    runs = [c.run(), c.run(room=0)]
    lost = 0.0
    for s, length in enumerate(lengths):
        k, v = c.cache.tokens(c.table[s], length)
        own = slice(c.start[s], c.start[s + 1])
        for head in range(2):
            of = slice(4 * head, 4 * head + 4)
            out, tol, lse, room = outputs(q[own, of], k[head], v[head], float(c.scale), t)
            for y, l in runs:
                off = np.abs(decode(y[own, of], t).astype(np.float64) - out)
                assert (off <= tol).all(), (s, head, np.max(off / tol))
                assert (np.abs(l[own, of] - lse) <= room).all(), (s, head)
            if head == 0:
                zero = outputs(q[own, of], 0 * k[0] if plane == "k" else k[0], 0 * v[0] if plane == "v" else v[0], float(c.scale), t)[0]
                lost += (np.abs(zero - out) > 2 * tol).mean() / len(lengths)
    assert lost > 0.8, lost
