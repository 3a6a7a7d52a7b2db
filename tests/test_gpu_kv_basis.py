"""Values written under the transform come out of the attention in the basis of a rotated bank: the append door, the attention and the output projection strung together on values that
four bits hold exactly in that basis."""
import ctypes as C

import numpy as np
import pytest

from oracle import qwkv
from oracle import qworacle as qo
from qwegn_amd import qwhip
from tests import helpers as H
from tests.test_gpu_heads import TYPES, decode, encode, np_type

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return qwhip.Device(0)


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("d,n", [(64, 1), (128, 5), (256, 23)])
def test_values_in_the_banks_basis(dev, d, n, t):
    """A token's block of values has one element, +- sqrt(32) and a little: under the transform all are +- 1 and as little, which the cache holds as +- 1 (a little less than 1 would be
    three quarters under the rule of the scale).  Equal weights (keys of zero), so the output's transform is the
    values' mean: an output is off by half a step and its weights by 2^-11 of their sizes, 1, an element of the transform by sqrt(32) times as much at most."""
    heads, shared, page, rng = 2, 3, 16, np.random.default_rng(d + n)
    v = np.zeros((n, heads, d // 32, 32), np.float32)
    for i in np.ndindex(v.shape[:3]):
        v[(*i, rng.integers(32))] = rng.choice([-1.0, 1.0]) * np.sqrt(32.0) * (1.0 + 2.0 ** -20)
    v = v.reshape(n, heads, d)
    pages = (n + page - 1) // page + 1
    kv = np.concatenate([np.zeros((n, heads * d), np.float32), v.reshape(n, -1)], 1)
    table = rng.permutation(pages)[: pages - 1].astype(np.int32).reshape(1, -1)
    slots = (table[0, np.arange(n) // page] * page + np.arange(n) % page).astype(np.int32)
    q = encode(rng.standard_normal((1, heads * shared, d)), t)
    room = qwkv.Cache(pages, page, heads, d, fill=0xFF)
    bufs = [dev.put(a) for a in (kv, slots, room.bytes, q, np.array([n], np.int32), table)]
    out, lib, st = dev.alloc(max(q.nbytes, 256)), dev.lib, dev.stream.handle
    view, batch = qwhip.KvCache(bufs[2].ptr, room.bytes.nbytes, pages, page, heads, d), qwhip.KvBatch(None, bufs[4].ptr, bufs[5].ptr, pages - 1, 1, 1, n)
    results = {}
    for flags in (qwhip.HEAD_FWHT_V, 0):
        rules = qwhip.HeadRules(flags=flags)
        qwhip.check(lib.qwhip_kv_append_mxfp4(st, C.byref(view), C.byref(rules), n, bufs[1].ptr, bufs[0].ptr, 2 * heads * d, bufs[0].ptr + 4 * heads * d, 2 * heads * d, qwhip.F32, None, 0, 0, None,
                                              0, 0, None, None))
        qwhip.check(lib.qwhip_kv_attention_mxfp4(st, C.byref(view), C.byref(batch), bufs[3].ptr, TYPES[t], heads * shared, 0, 1, d ** -0.5, 0, out.ptr, 0, None, None, 0))
        dev.stream.sync()
        results[flags] = out.download(np_type(t), (1, heads * shared, d))
    mean = np.repeat(v.astype(np.float64).mean(0), shared, 0)                             # [q_heads, d]
    off = 2.0 ** -11 * 1.01 + (2.0 ** -11 if t == "f16" else 2.0 ** -8)                   # of outputs up to 1
    turned = decode(results[qwhip.HEAD_FWHT_V], t).astype(np.float64)
    bound = np.sqrt(32.0) * (off + 2.0 ** -19)
    assert bound < 0.1 * np.abs(mean).max()
    assert (np.abs(qwkv.fwht32(turned)[0] - mean) <= bound).all()
    assert np.abs(turned[0] - mean).max() > 4 * bound                                     # another basis than the values'
    assert np.abs(decode(results[0], t)[0] - mean).max() < 0.07 * np.sqrt(32.0)           # which they come out in without the flag, to four bits
    if t == "f16":
        # a rotated bank takes the rows as they are
        blocks, w = H.make_bank("hq4_g64", 256, heads * shared * d, seed=3)
        bank, y = dev.put(blocks), dev.alloc(512)
        o = H.view_of(dev, bank, "hq4_g64", 256, heads * shared * d)
        qwhip.check(lib.qwhip_fill_u32(st, out.ptr, 0, out.nbytes // 4))
        out.upload(results[qwhip.HEAD_FWHT_V])
        qwhip.check(lib.qwhip_gemv(st, C.byref(o), out.ptr, qwhip.F16, 1, qwhip.X_PREROTATED, y.ptr, None))
        dev.stream.sync()
        want = qo.matmul_ref_f64(qwkv.fwht32(mean).reshape(1, -1), w)
        got = y.download(np.float16, (1, 256))
        assert qo.normalized_error(got, want) <= 2e-3 + off
        assert qo.normalized_error(got, qo.matmul_ref_f64(mean.reshape(1, -1), w)) > 0.1
        bank.free(), y.free()
    for b in (*bufs, out):
        b.free()
