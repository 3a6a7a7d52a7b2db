"""The definitions of oracle/qwkv.py against what pins them (CPU)."""
import numpy as np
import pytest

from oracle import qwkv, qwmx
from oracle import qworacle as qo


def test_transform_is_the_containers():
    x = np.random.default_rng(1).standard_normal((5, 3, 96)).astype(np.float32)
    assert np.array_equal(qwkv.fwht32(x), qo.fwht32_ortho(x.reshape(-1, 96)).reshape(x.shape))


@pytest.mark.parametrize("pairs", [False, True])
def test_rules_in_both_precisions(pairs):
    """The fp32 operations stay by the definition; a rotation keeps lengths; transformed queries and keys keep their products."""
    rng = np.random.default_rng(2)
    x, gamma = rng.standard_normal((7, 4, 64)), (1 + 0.1 * rng.standard_normal(64)).astype(np.float16)
    table, pos = qwkv.table(50, 32), rng.integers(0, 50, 7)
    a = qwkv.heads(x.astype(np.float32), gamma, False, 1e-6, table, pos, pairs, True)
    b = qwkv.heads(x.astype(np.float32), gamma, False, 1e-6, table, pos, pairs, True, np.float64)
    assert np.abs(a - b).max() <= 2.0 ** -18 * np.abs(b).max()
    turned = qwkv.heads(x, None, False, 0, table, pos, pairs, False, np.float64)
    assert np.allclose(np.linalg.norm(turned, axis=2), np.linalg.norm(x, axis=2), rtol=1e-6)   # the table is fp32
    assert np.array_equal(turned[..., 32:], x[..., 32:])
    q, k = rng.standard_normal((2, 3, 1, 64))
    assert np.allclose((qwkv.fwht32(q) * qwkv.fwht32(k)).sum(-1), (q * k).sum(-1))
    # a position outside the table takes its nearest row
    far = qwkv.heads(x, None, False, 0, table, np.full(7, 99), pairs, False, np.float64)
    assert np.array_equal(far, qwkv.heads(x, None, False, 0, table, np.full(7, 49), pairs, False, np.float64))


@pytest.mark.parametrize("page,d", [(16, 64), (32, 128), (256, 256)])
def test_pages_hold_what_is_put(page, d):
    rng = np.random.default_rng(3)
    c = qwkv.Cache(4, page, 3, d, fill=0x5A)
    before = c.bytes.copy()
    n = page + 5
    k, v = rng.standard_normal((2, n, 3, d)).astype(np.float32)
    table = [2, 0]
    t = np.arange(n)
    c.put(np.array(table)[t // page] * page + t % page, k, v)
    for got, x in zip(c.tokens(table, n), (k, v)):
        want = qwmx.values(*qwmx.quantise(x.reshape(-1, d))).reshape(n, 3, d).transpose(1, 0, 2)
        assert np.array_equal(got, want)
    assert np.array_equal(c.bytes[1], before[1]) and np.array_equal(c.bytes[3], before[3])
    c.put(np.array([-1, 4 * page]), k[:2], v[:2])                                        # left out
    assert np.array_equal(c.bytes[3], before[3])
    # the bytes of token 9, head 1, in the documented places
    codes, scales = qwmx.quantise(np.stack([k[9, 1], v[9, 1]]))
    piece, b = c.bytes[2, 1], page * d // 2
    assert np.array_equal(piece[9 * d // 2: 10 * d // 2], codes[0]) and np.array_equal(piece[b + 9 * d // 32: b + 10 * d // 32], scales[0])
    at = b + page * d // 32
    words = piece[at: at + b].reshape(page // 8, d // 8, 8, 4)
    assert np.array_equal(words[1, :, 1].reshape(-1), codes[1])
    assert np.array_equal(piece[at + b:].reshape(page // 8, d // 32, 8)[1, :, 1], scales[1])


def test_attention_definition():
    rng = np.random.default_rng(4)
    q, k, v = rng.standard_normal((6, 4, 64)), rng.standard_normal((2, 9, 64)), rng.standard_normal((2, 9, 64))
    out, lse, size = qwkv.attention(q, k, v, 0.125, window=3)
    i, h = 4, 3
    pos = 9 - 6 + i
    s = np.array([q[i, h] @ k[1, t] * 0.125 for t in range(pos - 2, pos + 1)])
    w = np.exp(s) / np.exp(s).sum()
    assert np.allclose(out[i, h], w @ v[1, pos - 2: pos + 1]) and np.isclose(lse[i, h], np.log(np.exp(s).sum())) and np.allclose(size[i, h], w @ np.abs(v[1, pos - 2: pos + 1]))
    out, lse, _ = qwkv.attention(q, k[:, :4], v[:, :4], 0.125)                            # two rows before the first token
    assert (out[:2] == 0).all() and (lse[:2] == -np.inf).all() and np.isfinite(lse[2:]).all()
    k[0, 8] = np.nan
    out, _, _ = qwkv.attention(q, k, v, 0.125)
    assert np.isnan(out[5, :2]).all() and np.isfinite(out[:5]).all() and np.isfinite(out[5, 2:]).all()
