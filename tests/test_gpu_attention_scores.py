"""qwhip_kv_attention_mxfp4 at the ends of what scores and weights can be, in the streaming and in the tile kernel: small weights beside a large one, scaled scores under
fp32's range and far from zero, values near fp32's range.

Bounds: half a step of the output's type, half a step of f16 (2^-11) of each weight, e = (D + 8) 2^-24 scale sum |q k| + 2^-20 of a score.  Where a weight
is subnormal in f16 half of that type's smallest step, 2^-25: weights stand at 2^12 and more under the maximum, so n of them are off by n 2^-37 max |v| of the sum."""
import numpy as np
import pytest

from oracle import qwkv
from qwegn_amd import qwhip
from tests.test_gpu_attention import HALF_STEP, Case
from tests.test_gpu_attention_tiles import Tiles
from tests.test_gpu_heads import decode, encode

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return qwhip.Device(0)


def fill(c, seq, k, v):
    """Keys and values [n, heads, d] as the tokens of a sequence."""
    t = np.arange(len(k))
    c.cache.put(c.table[seq][t // c.page] * c.page + t % c.page, np.asarray(k, np.float32), np.asarray(v, np.float32))


ROWS = [(Case, [1], 0), (Case, [1], 1 << 24), (Case, [9], 1 << 24), (Tiles, [64], 0), (Tiles, [64], 1 << 24)]


@pytest.mark.parametrize("cls,rows,room,d", [(*r, d) for r in ROWS for d in (64, 128, 256) if r[0] is Case or d < 256])
@pytest.mark.parametrize("t", ["f16", "bf16"])
def test_a_long_tail_behind_sinks_of_no_value(dev, cls, rows, room, d, t):
    """Four tokens whose values are zero hold nearly all of the weight, 16000 others lie 14, 16, 18 and 20 nats (up to 29 binary digits) below: the output is theirs."""
    n, rng = 16300, np.random.default_rng(d)
    c = cls(dev, 1, d, 1, 4, 64, rows, [n], t, scale=8.0 / d, noise=False)
    k, v = np.zeros((n, 1, d)), rng.uniform(0.5, 1.5, (n, 1, d))
    k[[0, 32, 64, 96]], v[[0, 32, 64, 96]] = 1.0, 0.0                                     # one for each of four ranges that interleave
    fill(c, 0, k, v)
    q = np.broadcast_to(np.array([1.75, 2.0, 2.25, 2.5])[None, :, None], (c.total, 4, d))
    c.q = encode(q, t)
    y, l = c.run(room=room)
    kk, vv = c.cache.tokens(c.table[0], n)
    want, lse, size = qwkv.attention(q[: rows[0]], kk, vv, 8.0 / d)
    e = (d + 8) * 2.0 ** -24 * 20.0 + 2.0 ** -20
    assert (want[:, 3].max() < 2.0 ** -11)                                                # what is there to be lost
    tol = HALF_STEP[t] * np.abs(want) + (2.0 ** -11 * 1.01 + 2 * e) * size + n * 2.0 ** -37 * vv.max() + 2.0 ** -25 * (t == "f16")
    off = np.abs(decode(y[: rows[0]], t).astype(np.float64) - want)
    assert (off <= tol).all(), (np.max(off / tol), np.max(off / want))
    assert (np.abs(l[: rows[0]] - lse) <= e + 2.0 ** -22 * (np.abs(lse) + np.log(n))).all()


@pytest.mark.parametrize("cls,rows,room", ROWS)
@pytest.mark.parametrize("t", ["f16", "bf16"])
def test_scaled_scores_under_the_range(dev, cls, rows, room, t):
    """Rows whose scaled scores are all under fp32's range have only scores of -inf: zeros and -inf, whatever the rows beside them have.  Rows with some of them
    have the others alone, rows with one over the range NaN."""
    n, d, scale = 3000, 64, 1.6e38
    c = cls(dev, 2, d, 1, 4, 32, rows, [n], t, scale=scale, noise=False)
    k = np.ones((n, 1, d))
    k[1::3] = 0.0
    v = np.random.default_rng(3).standard_normal((n, 1, d))
    fill(c, 0, k, v)
    q = np.zeros((c.total, 4, d))
    q[:, 0], q[:, 3] = -1.0, 0.0                                                          # zeros of the second kind: -64 1.6e38 or 0
    if rows[0] > 1:
        q[1:rows[0]:2, 3] = 1.0                                                           # over the range
    c.q = encode(q, t)
    half = np.ones((n, 1, d))                                                             # and once without a token of score zero
    for keys, low in ((k, False), (half, True)):
        fill(c, 0, keys, v)
        y, l = c.run(room=room)
        got = decode(y[: rows[0]], t).astype(np.float64)
        kk, vv = c.cache.tokens(c.table[0], n)
        for i in range(rows[0]):
            seen = n - rows[0] + i + 1
            for h in range(4):
                if q[i, h, 0] > 0:
                    assert np.isnan(got[i, h]).all() and np.isnan(l[i, h]), (i, h)
                elif q[i, h, 0] < 0 and low:
                    assert (got[i, h] == 0).all() and l[i, h] == -np.inf, (i, h)
                else:
                    own = np.arange(seen) % 3 == 1 if q[i, h, 0] < 0 else np.arange(seen) >= 0
                    x = vv[0, :seen][own]
                    tol = HALF_STEP[t] * np.abs(x.mean(0)) + 2.0 ** -11 * 1.01 * np.abs(x).mean(0) + 2.0 ** -25
                    assert (np.abs(got[i, h] - x.mean(0)) <= tol).all() and abs(l[i, h] - np.log(len(x))) <= 2.0 ** -18, (i, h)


@pytest.mark.parametrize("cls,rows,room", ROWS)
@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("scale", [2.0 ** 14, 2.0 ** 20 + 3.0, 1e8, 1e9, 3e12, 1e30])
def test_scores_far_from_zero(dev, cls, rows, room, t, scale):
    """Scaled scores of 2^14 .. 2^110, distinct ones far apart: a row's largest tokens share all of the weight, equal ones equally, and fp32's rounding of a score far
    from zero is no factor of the weight.  The products are exact in fp32 here, so that equal is equal."""
    n, d, heads, shared = 1900, 64, 2, 4
    c = cls(dev, 4, d, heads, shared, 16, rows, [n], t, scale=scale, noise=False)
    rng = np.random.default_rng(5)
    k = rng.standard_normal((n, heads, d))
    k = k[np.arange(n) % 41]                                                              # every key 46 times
    k[:, 1] = k[0, 1]                                                                     # the second head: one score, far over or under zero
    fill(c, 0, k, rng.standard_normal((n, heads, d)))
    q = rng.integers(-7, 8, (c.total, heads * shared, d)).astype(np.float64)
    c.q = encode(q, t)
    y, l = c.run(room=room)
    kk, vv = c.cache.tokens(c.table[0], n)
    for i in range(rows[0]):
        for h in range(heads * shared):
            seen = n - rows[0] + i + 1
            x = kk[h // shared, :seen] @ q[i, h]
            assert (x * 64 == np.round(x * 64)).all() and np.abs(kk[h // shared, 0]) @ np.abs(q[i, h]) < 2.0 ** 15   # exact in fp32
            best = x == x.max()
            assert best.all() or (x.max() - x[~best].max()) * scale > 200.0
            v = vv[h // shared, :seen][best]
            want, size, lse = v.mean(0), np.abs(v).mean(0), x.max() * scale + np.log(len(v))
            off = np.abs(decode(y[i, h], t).astype(np.float64) - want)
            assert (off <= HALF_STEP[t] * np.abs(want) + 2.0 ** -11 * 1.01 * size + 2.0 ** -25).all(), (i, h, x.max())
            assert abs(l[i, h] - lse) <= 2.0 ** -21 * abs(lse) + 2.0 ** -18, (i, h)


@pytest.mark.parametrize("cls,rows,room", ROWS)
def test_values_near_the_range_of_fp32(dev, cls, rows, room):
    """Values of 2^125 and scores that grow by less than eight binary digits: a weight is at most one then, and no sum leaves fp32's range that the result does not leave."""
    n, d = 1500, 64
    c = cls(dev, 6, d, 1, 4, 16, rows, [n], "bf16", scale=1.0 / 8.0, noise=False)
    t = np.arange(n)
    k = np.zeros((n, 1, d))
    k[:, 0, 0] = np.where(t == 700, 4.0, np.where(t == 1300, 6.0, 0.0))                   # 0, 3.25 and 4.875 nats
    fill(c, 0, k, np.zeros((n, 1, d)))
    kc, ks, vc, vs = c.cache.planes()
    rng = np.random.default_rng(7)
    v = np.where(np.isin(t, (5, 700, 1300))[:, None], 1.0, 0.0) * np.where(rng.random((1, d)) < 0.5, 1.0, -1.0)
    fill(c, 0, k, v[:, None] * 4.0)                                                       # elements of 4 under a byte of 127 ..
    for s in (5, 700, 1300):
        p, o = c.table[0][s // 16], s % 16
        assert (vs[p, 0, o // 8, :, o % 8] == 127).all()
        vs[p, 0, o // 8, :, o % 8] = 250                                                  # .. of 250: 2^125
    q = np.zeros((c.total, 4, d))
    q[..., 0] = 6.5
    c.q = encode(q, "bf16")
    y, l = c.run(room=room)
    kk, vv = c.cache.tokens(c.table[0], n)
    want, lse, size = qwkv.attention(q[: rows[0]], kk, vv, 1.0 / 8.0)
    got = decode(y[: rows[0]], "bf16").astype(np.float64)
    assert np.isfinite(want).all() and np.abs(want).min() > 2.0 ** 115
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + (2.0 ** -11 + 2.0 ** -16) * size).all()
    assert (np.abs(l[: rows[0]] - lse) <= 2.0 ** -18).all()


@pytest.mark.parametrize("cls,rows,room", ROWS)
@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("scale", [128.0 ** -0.5, 0.3, 7.1, 1e-6])
def test_the_logarithm_has_the_precision_of_fp32(dev, cls, rows, room, t, scale):
    """One token decides (the others lie 30 nats or more below, which fp32's one does not notice) or all do, with a product that is exact in fp32: the logarithm is off by a rounding of a
    score, one of its own (2^-24 each) and 2^-20 for the exponents of the weights."""
    n, d = 1700, 64
    c = cls(dev, 8, d, 1, 4, 32, rows, [n], t, scale=scale, noise=False)
    rng = np.random.default_rng(9)
    k = np.zeros((n, 1, d))
    k[0] = rng.choice([1.0, 1.5, 2.0, 3.0, 4.0], d)                                       # the first token is seen by all rows
    fill(c, 0, k, rng.standard_normal((n, 1, d)))
    q = rng.integers(1, 60, (c.total, 4, d)).astype(np.float64)
    q[:, 3] = 0.0
    c.q = encode(q, t)
    y, l = c.run(room=room)
    kk, _ = c.cache.tokens(c.table[0], n)
    for i in range(rows[0]):
        seen = n - rows[0] + i + 1
        for h in range(4):
            x = float(q[i, h] @ kk[0, 0]) * float(np.float32(scale))
            want = np.logaddexp(x, np.log(seen - 1.0))
            assert abs(l[i, h] - want) <= 2.0 ** -23 * abs(want) + 2.0 ** -20, (i, h, l[i, h], want)
