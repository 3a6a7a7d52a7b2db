"""qwhip_head_norm_rope and qwhip_kv_append_mxfp4 against their fp32 definition, bit for bit: every operation of the doors is rounded by itself and in a
given order, so the tolerance is zero (and the definition is within 2^-18 of the one in 64 bits, which is checked here too)."""
import ctypes as C

import numpy as np
import pytest

from oracle import qwkv
from oracle import qworacle as qo
from qwegn_amd import qwhip

pytestmark = pytest.mark.gpu
TYPES = {"f32": qwhip.F32, "f16": qwhip.F16, "bf16": qwhip.BF16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


@pytest.fixture(scope="module")
def dev():
    return qwhip.Device(0)


def encode(x, t):
    """f32 -> the type's bits."""
    return x.astype(np.float32) if t == "f32" else x.astype(np.float16) if t == "f16" else qo.f32_to_bf16_bits(x.astype(np.float32))


def decode(b, t):
    return qo.bf16_bits_to_f32(b) if t == "bf16" else b.astype(np.float32)


def same(got, want, t):
    """Bits, with any NaN equal to any other."""
    a, b = decode(got, t), decode(want, t)
    nan = np.isnan(a) & np.isnan(b)
    return np.array_equal(np.where(nan, 0, got.view(np.uint32 if t == "f32" else np.uint16)), np.where(nan, 0, want.view(np.uint32 if t == "f32" else np.uint16)))


def np_type(t):
    return {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}[t]


class Rules:
    def __init__(self, dev, rng, d, rows, rope=0, flags=0, q=True, k=True, positions=700):
        self.flags, self.d, self.rope, self.keep = flags, d, rope, []
        centre = 0.0 if flags & qwkv.PLUS_ONE else 1.0
        self.gamma = {n: (centre + 0.2 * rng.standard_normal(d)).astype(np.float16) if on else None for n, on in (("q", q), ("k", k))}
        self.table = qwkv.table(positions, rope) if rope else None
        self.position = rng.integers(-3, positions + 3, rows).astype(np.int32)            # some outside the table

        def put(a):
            if a is None:
                return None
            self.keep.append(dev.put(a))
            return self.keep[-1].ptr

        self.c = qwhip.HeadRules(position=put(self.position), cos_sin=put(self.table), q_gamma=put(self.gamma["q"]), k_gamma=put(self.gamma["k"]), positions=positions,
                                 rope_dims=rope, eps=1e-6, flags=flags)

    def of(self, x, side, dtype=np.float32):
        if side == "v":
            return qwkv.heads(x, fwht=bool(self.flags & qwkv.FWHT_V), dtype=dtype)
        return qwkv.heads(x, self.gamma[side], bool(self.flags & qwkv.PLUS_ONE), 1e-6, self.table, self.position, bool(self.flags & qwkv.PAIRS), bool(self.flags & qwkv.FWHT_QK), dtype)

    def free(self):
        for b in self.keep:
            b.free()


def run_norm_rope(dev, rules, x, rows, d, qh, kh, ld, t, o, ldqo=0, ldko=0, stream=None):
    """x: bits [rows, ld], queries first, keys behind them."""
    xb = dev.put(x)
    ldqo, ldko = ldqo or qh * d, ldko or kh * d
    qb, kb = dev.alloc(max(rows * ldqo * SIZE[o], 256)), dev.alloc(max(rows * ldko * SIZE[o], 256))
    st = stream or dev.stream
    for b, n in ((qb, rows * ldqo), (kb, rows * ldko)):
        qwhip.check(dev.lib.qwhip_fill_u32(st.handle, b.ptr, 0x7E017E01, b.nbytes // 4))
    qwhip.check(dev.lib.qwhip_head_norm_rope(st.handle, C.byref(rules.c), rows, d, xb.ptr, qh, ld, xb.ptr + qh * d * SIZE[t], kh, ld, TYPES[t], qb.ptr, ldqo, kb.ptr, ldko, TYPES[o]))
    st.sync()
    q, k = qb.download(np_type(o), (rows, ldqo)), kb.download(np_type(o), (rows, ldko))
    for b in (xb, qb, kb):
        b.free()
    return q, k


@pytest.mark.parametrize("rows,d,qh,kh,rope,flags,t,o", [
    (1, 128, 40, 8, 128, qwkv.PLUS_ONE, "f16", "f16"),
    (1, 32, 1, 1, 0, 0, "bf16", "f32"),
    (3, 32, 3, 1, 32, qwkv.FWHT_QK, "f32", "bf16"),
    (5, 64, 4, 1, 32, qwkv.PAIRS | qwkv.PLUS_ONE, "bf16", "bf16"),
    (333, 96, 6, 3, 48, qwkv.PAIRS | qwkv.FWHT_QK, "f32", "bf16"),
    (17, 96, 5, 0, 96, 0, "f16", "f32"),
    (9, 160, 2, 2, 16, qwkv.FWHT_QK, "bf16", "f16"),
    (13, 192, 0, 7, 192, qwkv.PLUS_ONE, "f32", "f32"),
    (31, 224, 3, 1, 112, 0, "f16", "f16"),
    (257, 256, 16, 2, 64, qwkv.PLUS_ONE | qwkv.FWHT_QK, "bf16", "bf16"),
    (2500, 64, 9, 1, 64, qwkv.FWHT_QK, "f16", "f16"),          # rows whose heads one workgroup walks over
    (2049, 128, 40, 8, 128, 0, "bf16", "bf16"),
])
def test_norm_rope(dev, rows, d, qh, kh, rope, flags, t, o):
    rng = np.random.default_rng(rows * d + qh)
    rules = Rules(dev, rng, d, rows, rope, flags)
    ld = (qh + kh) * d + 24
    x = encode(rng.standard_normal((rows, ld)) * np.exp(rng.standard_normal((rows, 1)) * 3), t)
    q, k = run_norm_rope(dev, rules, x, rows, d, qh, kh, ld, t, o, ldko=kh * d + 8)
    val = decode(x, t)
    assert (k[:, kh * d:] == (np.float32(np.array(0x7E017E01, np.uint32).view(np.float32)) if o == "f32" else np.array(0x7E01, np.uint16).view(np_type(o)) if o == "f16" else 0x7E01)).all() or \
        np.isnan(decode(k[:, kh * d:], o)).all()
    for got, n, off, side in ((q, qh, 0, "q"), (k[:, : kh * d], kh, qh * d, "k")):
        part = val[:, off:off + n * d].reshape(rows, n, d)
        want = rules.of(part, side)
        assert same(np.ascontiguousarray(got).reshape(rows, n, d), encode(want, o), o), side
        wide = rules.of(part, side, np.float64)
        if n:
            # against the definition: at most 2 D roundings of relative 2^-24 each on numbers no larger than the head's (sqrt(2 D) of them after the transform)
            bound = 2.0 ** -18 * np.linalg.norm(wide, axis=2, keepdims=True) + 1e-30
            assert (np.abs(want - wide) <= bound).all()
    rules.free()


@pytest.mark.parametrize("t", ["f16", "f32"])
def test_in_place_without_norm_or_rotation(dev, t):
    rows, d, qh, kh = 700, 128, 5, 3
    rng = np.random.default_rng(5)
    for rope, q_on, flags in ((128, True, qwkv.PLUS_ONE), (64, False, qwkv.PAIRS), (0, False, qwkv.FWHT_QK)):
        rules = Rules(dev, rng, d, rows, rope, flags, q=q_on, k=False)
        ld = (qh + kh + 2) * d
        x = encode(rng.standard_normal((rows, ld)), t)
        xb = dev.put(x)
        k = xb.ptr + qh * d * SIZE[t]
        qwhip.check(dev.lib.qwhip_head_norm_rope(dev.stream.handle, C.byref(rules.c), rows, d, xb.ptr, qh, ld, k, kh, ld, TYPES[t], xb.ptr, ld, k, ld, TYPES[t]))
        dev.stream.sync()
        got, val = xb.download(np_type(t), x.shape), decode(x, t)
        for side, off, n in (("q", 0, qh), ("k", qh, kh)):
            want = rules.of(val[:, off * d:(off + n) * d].reshape(rows, n, d), side)
            assert same(np.ascontiguousarray(got[:, off * d:(off + n) * d]).reshape(rows, n, d), encode(want, t), t)
        assert np.array_equal(got[:, (qh + kh) * d:], x[:, (qh + kh) * d:])
        xb.free()
        rules.free()


def test_zeros_infinities_and_nan_stay_in_their_head(dev):
    rows, d, qh, kh = 6, 64, 3, 2
    rng = np.random.default_rng(8)
    rules = Rules(dev, rng, d, rows, 32, qwkv.FWHT_QK)
    x = rng.standard_normal((rows, (qh + kh) * d)).astype(np.float32)
    x[0, :d] = 0.0
    x[1, d + 5], x[2, 3 * d + 40], x[3, 2 * d] = np.inf, np.nan, 3e38
    x[4, :d] = 1e-30
    x = encode(x, "f32")
    q, k = run_norm_rope(dev, rules, x, rows, d, qh, kh, (qh + kh) * d, "f32", "f32")
    with np.errstate(all="ignore"):
        assert same(q.reshape(rows, qh, d), rules.of(x[:, :qh * d].reshape(rows, qh, d), "q"), "f32")
        assert same(k.reshape(rows, kh, d), rules.of(x[:, qh * d:].reshape(rows, kh, d), "k"), "f32")
    rules.free()


def run_append(dev, cache, rules, x, slots, rows, qh, t, o, values=True, ld=None, stream=None):
    """x: bits [rows, ld], queries, keys, values.  Returns (pages, q_out, k_values, v_values)."""
    kh, d, st = cache.heads, cache.d, stream or dev.stream
    ld = ld or (qh + 2 * kh) * d
    xb, sb, pb = dev.put(x), dev.put(slots), dev.put(cache.bytes)
    outs = [dev.alloc(max(rows * n * d * SIZE[o], 256)) for n in (qh, kh, kh)]
    for b in outs:
        qwhip.check(dev.lib.qwhip_fill_u32(st.handle, b.ptr, 0x7E017E01, b.nbytes // 4))
    view = qwhip.KvCache(pb.ptr, cache.bytes.nbytes, len(cache.bytes), cache.page, kh, d)
    k = xb.ptr + qh * d * SIZE[t]
    qwhip.check(dev.lib.qwhip_kv_append_mxfp4(st.handle, C.byref(view), C.byref(rules.c) if rules else None, rows, sb.ptr, k, ld, k + kh * d * SIZE[t], ld, TYPES[t], xb.ptr, qh, ld,
                                              outs[0].ptr, 0, TYPES[o], outs[1].ptr if values else None, outs[2].ptr if values else None))
    st.sync()
    pages = pb.download(np.uint8, cache.bytes.shape)
    res = [b.download(np_type(o), (rows, n, d)) for b, n in zip(outs, (qh, kh, kh))]
    for b in (xb, sb, pb, *outs):
        b.free()
    return pages, *res


def check_append(cache, rules, x, slots, rows, qh, t, o, got, values=True, ld=None):
    kh, d = cache.heads, cache.d
    pages, q, kv, vv = got
    val = decode(x, t)[:, : (qh + 2 * kh) * d].reshape(rows, -1, d)
    with np.errstate(all="ignore"):
        sides = [rules.of(val[:, a:b], n) if rules else val[:, a:b] for n, a, b in (("q", 0, qh), ("k", qh, qh + kh), ("v", qh + kh, qh + 2 * kh))]
    cache.put(slots, sides[1], sides[2])
    assert np.array_equal(pages, cache.bytes)
    there = (slots >= 0) & (slots < len(cache.bytes) * cache.page)
    untouched = np.full(2, 0x7E01, np.uint16)
    if qh:
        assert same(q[there], encode(sides[0], o)[there], o)
    for a in ([q] if qh else []) + [kv, vv]:
        rest = a[~there].view(np.uint16)
        assert (rest == untouched[0]).all()
    if values:
        from oracle import qwmx
        for a, side in ((kv, sides[1]), (vv, sides[2])):
            c, s = qwmx.quantise(side.reshape(-1, d))
            assert same(a[there], encode(qwmx.values(c, s).reshape(rows, kh, d).astype(np.float32), o)[there], o)
    else:
        assert (kv.view(np.uint16) == untouched[0]).all() and (vv.view(np.uint16) == untouched[0]).all()


@pytest.mark.parametrize("rows,d,qh,kh,page,rope,flags,t,o", [
    (1, 128, 40, 8, 64, 128, qwkv.PLUS_ONE | qwkv.FWHT_QK | qwkv.FWHT_V, "f16", "f16"),
    (250, 256, 16, 2, 16, 64, qwkv.PLUS_ONE, "bf16", "bf16"),
    (7, 64, 0, 1, 16, 0, 0, "f32", "f16"),
    (40, 64, 6, 3, 32, 64, qwkv.PAIRS | qwkv.FWHT_V, "f32", "f32"),
    (129, 128, 4, 4, 256, 32, qwkv.FWHT_QK, "bf16", "f32"),
    (2100, 128, 2, 2, 128, 128, qwkv.FWHT_QK | qwkv.FWHT_V, "bf16", "bf16"),
])
def test_append(dev, rows, d, qh, kh, page, rope, flags, t, o):
    rng = np.random.default_rng(rows + d)
    cache = qwkv.Cache((rows + 60) // page + 2, page, kh, d)
    cache.bytes[:] = rng.integers(0, 256, cache.bytes.shape)                              # what no row names stays
    slots = rng.permutation(len(cache.bytes) * page)[:rows].astype(np.int32)
    if rows > 5:
        slots[2], slots[4], slots[5] = -1, -2 ** 31, len(cache.bytes) * page
    ld = (qh + 2 * kh) * d + 8
    rules = Rules(dev, rng, d, rows, rope, flags, k=rows % 2 == 0)
    x = encode(rng.standard_normal((rows, ld)) * np.exp(rng.standard_normal((rows, 1))), t)
    got = run_append(dev, cache, rules, x, slots, rows, qh, t, o, ld=ld)
    check_append(cache, rules, x, slots, rows, qh, t, o, got)
    rules.free()


def test_append_plain_zeros_broken_blocks_and_extremes(dev):
    """No rules and no values; blocks of zeros, with infinities and NaN, of subnormal and of the largest numbers."""
    rows, d, kh = 24, 64, 2
    rng = np.random.default_rng(9)
    cache = qwkv.Cache(3, 16, kh, d, fill=0xAB)
    x = rng.standard_normal((rows, 2 * kh * d)).astype(np.float32)
    x[0], x[1, 7], x[2, 40], x[3, 200] = 0.0, np.inf, np.nan, -np.inf
    x[4], x[5] = x[4] * 1e-40, np.clip(x[5], -1.0, 1.0) * 3.4e38
    slots = rng.permutation(48)[:rows].astype(np.int32)
    got = run_append(dev, cache, None, x, slots, rows, 0, "f32", "f32", values=False)
    check_append(cache, None, x, slots, rows, 0, "f32", "f32", got, values=False)


def test_append_as_norm_rope_and_at_every_number_of_rows(dev):
    """A row's bits do not depend on the door nor on the rows beside it."""
    d, qh, kh, page, rows = 128, 8, 2, 16, 2300
    rng = np.random.default_rng(10)
    rules = Rules(dev, rng, d, rows, 128, qwkv.PLUS_ONE | qwkv.FWHT_QK)
    x = encode(rng.standard_normal((rows, (qh + 2 * kh) * d)), "bf16")
    cache = qwkv.Cache(rows // page + 1, page, kh, d)
    slots = np.arange(rows, dtype=np.int32)
    pages, q, kv, _ = run_append(dev, cache, rules, x, slots, rows, qh, "bf16", "bf16")
    q2, _ = run_norm_rope(dev, rules, x, rows, d, qh, kh, x.shape[1], "bf16", "bf16")
    assert np.array_equal(q2.reshape(q.shape), q)
    few = 19
    p3, q3, kv3, _ = run_append(dev, cache, rules, x[:few], slots[:few], few, qh, "bf16", "bf16")
    assert np.array_equal(q3, q[:few]) and np.array_equal(kv3, kv[:few]) and np.array_equal(p3[0], pages[0])
    rules.free()


def test_captured_and_on_two_streams(dev):
    d, qh, kh, page, rows = 64, 4, 2, 32, 50
    rng = np.random.default_rng(12)
    rules = Rules(dev, rng, d, rows, 64, qwkv.FWHT_V)
    st = qwhip.Stream(dev)
    xs = [encode(rng.standard_normal((rows, (qh + 2 * kh) * d)), "f16") for _ in range(3)]
    xb, pb, qb = dev.put(xs[0]), dev.put(qwkv.Cache(4, page, kh, d).bytes), dev.alloc(rows * qh * d * 2)
    slots = rng.permutation(128)[:rows].astype(np.int32)
    sb = dev.put(slots)
    view = qwhip.KvCache(pb.ptr, pb.nbytes, 4, page, kh, d)
    view.bytes = 4 * dev.lib.qwhip_kv_page_bytes(page, kh, d)

    def step():
        k = xb.ptr + qh * d * 2
        qwhip.check(dev.lib.qwhip_kv_append_mxfp4(st.handle, C.byref(view), C.byref(rules.c), rows, sb.ptr, k, (qh + 2 * kh) * d, k + kh * d * 2, (qh + 2 * kh) * d, qwhip.F16, xb.ptr, qh,
                                                  (qh + 2 * kh) * d, qb.ptr, 0, qwhip.F16, None, None))

    graph = qwhip.Graph(st, step)
    for x in xs:
        xb.upload(x)
        graph.launch()
        st.sync()
        cache = qwkv.Cache(4, page, kh, d)
        want = run_append(dev, cache, rules, x, slots, rows, qh, "f16", "f16")           # the other stream, eager
        assert np.array_equal(pb.download(np.uint8, cache.bytes.shape), want[0]) and np.array_equal(qb.download(np.float16, want[1].shape), want[1])
    graph.destroy()
    for b in (xb, pb, qb, sb):
        b.free()
    rules.free()


def test_append_with_queries_in_place_and_pitches(dev):
    """A projection's rows as they are: queries turned in place, keys and values out of the same rows."""
    d, qh, kh, page = 64, 6, 2, 16
    for rows in (30, 2200):
        rng = np.random.default_rng(rows)
        rules = Rules(dev, rng, d, rows, 64, qwkv.PLUS_ONE | qwkv.FWHT_QK | qwkv.FWHT_V)
        ld = (qh + 2 * kh) * d + 16
        x = encode(rng.standard_normal((rows, ld)), "f16")
        cache = qwkv.Cache(rows // page + 2, page, kh, d)
        slots = rng.permutation(len(cache.bytes) * page)[:rows].astype(np.int32)
        xb, sb, pb = dev.put(x), dev.put(slots), dev.put(cache.bytes)
        view = qwhip.KvCache(pb.ptr, cache.bytes.nbytes, len(cache.bytes), page, kh, d)
        k = xb.ptr + qh * d * 2
        qwhip.check(dev.lib.qwhip_kv_append_mxfp4(dev.stream.handle, C.byref(view), C.byref(rules.c), rows, sb.ptr, k, ld, k + kh * d * 2, ld, qwhip.F16, xb.ptr, qh, ld, xb.ptr, ld,
                                                  qwhip.F16, None, None))
        dev.stream.sync()
        val, got = decode(x, "f16"), xb.download(np.float16, x.shape)
        part = lambda a, n: val[:, a * d:(a + n) * d].reshape(rows, n, d)  # noqa: E731
        assert same(np.ascontiguousarray(got[:, : qh * d]).reshape(rows, qh, d), encode(rules.of(part(0, qh), "q"), "f16"), "f16")
        assert np.array_equal(got[:, qh * d:], x[:, qh * d:])
        cache.put(slots, rules.of(part(qh, kh), "k"), rules.of(part(qh + kh, kh), "v"))
        assert np.array_equal(pb.download(np.uint8, cache.bytes.shape), cache.bytes)
        for b in (xb, sb, pb):
            b.free()
        rules.free()
