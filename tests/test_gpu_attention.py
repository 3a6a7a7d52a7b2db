"""qwhip_kv_attention_mxfp4 against the definition in 64 bits, over caches that hold other things around what the rows see.

Bound of an output: half a step of its type; each weight's rounding to f16 in front of the product with the values (half a step, 2^-11 of it; 2^-25 of the
largest where it is subnormal), hence 2^-11 sum p |v| + L 2^-25 max |v|; and the score's error e = (D + 8) 2^-24 scale sum |q k| + 2^-20 (fp32 sums of exact
products, the exponent's own rounding), which moves weight and sum: 2 e sum p |v|.  The logarithm of the sum is off by e and its own rounding."""
import ctypes as C

import numpy as np
import pytest

from oracle import qwkv
from oracle import qworacle as qo
from qwegn_amd import qwhip
from tests.test_gpu_heads import TYPES, decode, encode, np_type

pytestmark = pytest.mark.gpu
HALF_STEP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}


@pytest.fixture(scope="module")
def dev():
    return qwhip.Device(0)


def bits(*pairs):
    return all(np.array_equal(a.view(np.uint8), b.view(np.uint8)) for a, b in pairs)


class Case:
    """Sequences of given rows and lengths over a cache that is otherwise noise."""

    def __init__(self, dev, seed, d, heads, shared, page, rows, lengths, t="f16", window=0, std=1.5, noise=True, scale=None):
        rng = np.random.default_rng(seed)
        self.dev, self.d, self.heads, self.shared, self.page, self.t, self.window = dev, d, heads, shared, page, t, window
        self.rows, self.lengths, self.seqs = np.array(rows), np.array(lengths), len(rows)
        self.scale = np.float32(d ** -0.5 if scale is None else scale)
        self.start = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        self.total = int(self.start[-1]) + 2                                              # two rows of padding
        self.each = max(1, int(-(-max(lengths) // page)))
        count = self.seqs * self.each + 3
        self.cache = qwkv.Cache(count, page, heads, d)
        if noise:
            self.cache.bytes[:] = rng.integers(0, 256, self.cache.bytes.shape)            # scale bytes of 255 and 0 among it
        self.table = rng.permutation(count)[: self.seqs * self.each].astype(np.int32).reshape(self.seqs, self.each)
        for s, n in enumerate(lengths):
            k, v = rng.standard_normal((2, n, heads, d)) * np.exp(0.5 * rng.standard_normal((2, n, 1, 1)))
            t_ = np.arange(n)
            self.cache.put(self.table[s][t_ // page] * page + t_ % page, k.astype(np.float32), v.astype(np.float32))
        self.q = encode(rng.standard_normal((self.total, heads * shared, d)) * std, t)

    def run(self, room=1 << 24, lse=True, stream=None, max_rows=None, max_length=None, ld=0, table=None, start=True):
        dev, st, heads = self.dev, stream or self.dev.stream, self.heads * self.shared
        ld = ld or heads * self.d
        q = np.zeros((self.total, ld), self.q.dtype)
        q[:, : heads * self.d] = self.q.reshape(self.total, -1)
        bufs = [dev.put(a) for a in (q, self.cache.bytes, self.start, self.lengths.astype(np.int32), self.table if table is None else table)]
        out, le, ws = dev.alloc(self.total * ld * 2), dev.alloc(self.total * heads * 4), dev.alloc(max(room, 256))
        for b in (out, le, ws):
            qwhip.check(dev.lib.qwhip_fill_u32(st.handle, b.ptr, 0x7E017E01, b.nbytes // 4))
        view = qwhip.KvCache(bufs[1].ptr, self.cache.bytes.nbytes, len(self.cache.bytes), self.page, self.heads, self.d)
        batch = qwhip.KvBatch(bufs[2].ptr if start else None, bufs[3].ptr, bufs[4].ptr, self.table.shape[1], self.seqs, int(max(self.rows)) if max_rows is None else max_rows,
                              int(max(self.lengths)) if max_length is None else max_length)
        rows = self.total if start else self.seqs
        self.need = dev.lib.qwhip_kv_attention_workspace_bytes(C.byref(view), C.byref(batch), heads, rows, self.window)
        qwhip.check(dev.lib.qwhip_kv_attention_mxfp4(st.handle, C.byref(view), C.byref(batch), bufs[0].ptr, TYPES[self.t], heads, ld, rows, self.scale, self.window, out.ptr, ld,
                                                     le.ptr if lse else None, ws.ptr if room else None, room))
        st.sync()
        y, l = out.download(np_type(self.t), (self.total, ld)), le.download(np.float32, (self.total, heads))
        for b in (*bufs, out, le, ws):
            b.free()
        pad = y[:, heads * self.d:]
        assert (pad.view(np.uint16) == 0x7E01).all()
        return np.ascontiguousarray(y[:, : heads * self.d]).reshape(self.q.shape), l

    def check(self, y, l):
        q = decode(self.q, self.t).astype(np.float64)
        u = HALF_STEP[self.t]
        for s in range(self.seqs):
            a, b, n = self.start[s], self.start[s + 1], int(self.lengths[s])
            if a == b:
                continue
            k, v = self.cache.tokens(self.table[s], n)
            want, lse, size = qwkv.attention(q[a:b], k, v, float(self.scale), self.window)
            kk = np.repeat(np.abs(np.nan_to_num(k, posinf=0, neginf=0)), self.shared, 0)
            reach = np.max(np.einsum("ihd,htd->iht", np.abs(q[a:b]), kk), axis=2, initial=0.0) * float(self.scale)
            e = (self.d + 8) * 2.0 ** -24 * reach + 2.0 ** -20
            top = np.max(np.abs(np.nan_to_num(v)), initial=0.0)
            tol = u * np.abs(want) + (2.0 ** -11 * 1.01 + 2 * e[..., None]) * size + n * 2.0 ** -25 * top + 2.0 ** -25
            got = decode(y[a:b], self.t).astype(np.float64)
            nan = np.isnan(want)
            assert np.array_equal(np.isnan(got), nan), s
            assert (np.abs(got - want)[~nan] <= tol[~nan]).all(), (s, np.nanmax(np.abs(got - want) / tol))
            fine = np.isfinite(lse)
            assert np.array_equal(l[a:b][~fine], lse[~fine].astype(np.float32), equal_nan=True)
            assert (np.abs(l[a:b][fine] - lse[fine]) <= (e + 2.0 ** -22 * (np.abs(lse) + np.log(n + 2.0)))[fine]).all(), s
        rest = slice(self.start[-1], self.total)
        assert (y[rest].view(np.uint16) == 0x7E01).all() and (l[rest].view(np.uint32) == 0x7E017E01).all()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("t", ["f16", "bf16"])
def test_tokens_of_all_lengths(dev, d, t):
    lengths = [1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 500, 0, 1111]
    c = Case(dev, d, d, 2, 5, 16, [1] * len(lengths), lengths, t)
    c.check(*c.run())


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("heads,shared", [(1, 1), (3, 2), (2, 16), (1, 23)])
def test_pages_and_groups(dev, page, heads, shared):
    c = Case(dev, page + shared, 64, heads, shared, page, [1, 3, 2], [300, 77, 513], "bf16")
    c.check(*c.run())


@pytest.mark.parametrize("d,t,window", [(64, "f16", 0), (128, "bf16", 0), (256, "f16", 0), (128, "f16", 1), (64, "bf16", 33), (256, "bf16", 100), (128, "bf16", 5000)])
def test_rows_of_ragged_sequences(dev, d, t, window):
    """Prompts from their first token, chunks behind cached tokens, a sequence without rows, one with more rows than tokens (rows that see nothing)."""
    c = Case(dev, d + window, d, 2, 3, 32, [70, 1, 0, 16, 45, 9, 200], [70, 200, 50, 321, 45, 4, 777], t, window)
    y, l = c.run()
    c.check(y, l)
    empty = slice(c.start[5], c.start[5] + 5)
    assert (decode(y[empty], t) == 0).all() and (l[empty] == -np.inf).all()


@pytest.mark.parametrize("rows", [[1], [16], [17], [40], [129], [300], [1000]])
@pytest.mark.parametrize("room", [0, 1 << 24])
def test_rows_of_one_sequence(dev, rows, room):
    c = Case(dev, rows[0], 128, 1, 4, 64, rows, [1500], "bf16")
    c.check(*c.run(room=room))


def test_room_gives_parts_and_little_room_few(dev):
    c = Case(dev, 3, 64, 2, 4, 16, [1], [40000], "f16", std=3.0)
    y0, l0 = c.run(room=0)
    c.check(y0, l0)
    y1, l1 = c.run()
    assert c.need > 0
    c.check(y1, l1)
    for room in (c.need, c.need // 3, 5000):
        y, l = c.run(room=room)
        c.check(y, l)
        if room == c.need:
            assert bits((y, y1), (l, l1))                        # more room than that changes nothing
    y, l = c.run()
    assert bits((y, y1), (l, l1))                                # the same call, the same bits


def test_peaked_and_flat_scores(dev):
    for std, scale in ((30.0, None), (1e-3, None), (1.0, 4.0), (1.0, 1e-4)):
        for t in ("f16", "bf16"):
            c = Case(dev, 17, 128, 1, 4, 16, [3, 1], [600, 900], t, std=std, scale=scale)
            c.check(*c.run())


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_scales_outside_of_the_half_types(dev, d, t):
    """Keys and values far above and below f16's range among ordinary ones, blocks of zeros."""
    c = Case(dev, 21, d, 2, 4, 16, [1, 20, 5], [200, 333, 64], t, std=0.3)
    kc, ks, vc, vs = c.cache.planes()
    rng = np.random.default_rng(4)
    ks[rng.random(ks.shape) < 0.02] = 100                                                 # 2^-27: q . k hardly notices, zero would be wrong
    vs[rng.random(vs.shape) < 0.02] = 100
    vs[rng.random(vs.shape) < 0.01] = 150                                                 # 2^23
    ks[rng.random(ks.shape) < 0.01] = 0
    vs[rng.random(vs.shape) < 0.01] = 1
    if t == "f16":
        vs[vs == 150] = 137                                                               # within the output's range
        ks[rng.random(ks.shape) < 0.001] = 143                                            # 2^16: past f16
    y, l = c.run()
    c.check(y, l)


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_broken_blocks_reach_the_rows_that_see_them_only(dev, d, t):
    c = Case(dev, 33, d, 2, 3, 16, [40, 1, 1], [100, 300, 90], t)
    kc, ks, vc, vs = c.cache.planes()

    def at(seq, token):
        return c.table[seq][token // 16], token % 16

    p, o = at(0, 80)
    vs[p, 1, o // 8, 1, o % 8] = 255                                                      # rows 20 .. of sequence 0, head 1, elements 32 .. 63
    p, o = at(0, 90)
    ks[p, 0, o, 0] = 255                                                                  # rows 30 .., head 0: all elements
    p, o = at(1, 5)
    vs[p, 0, o // 8, d // 32 - 1, o % 8] = 255
    y, l = c.run()
    c.check(y, l)
    got = decode(y, t)
    assert np.isnan(got[20:40, 3:, 32:64]).all() and np.isfinite(got[:20, 3:]).all() and np.isfinite(got[20:30, :3]).all() and np.isnan(got[30:40, :3]).all()
    # and infinities and NaN of a query stay in its row and head
    c = Case(dev, 34, d, 2, 3, 16, [5, 1], [50, 200], t)
    x = decode(c.q, t).astype(np.float32)
    x[1, 2, 7], x[5, 0, 1] = np.nan, np.nan
    c.q = encode(x, t)
    c.check(*c.run())


def test_window_over_freed_pages(dev):
    """Pages behind the window may be gone from the table."""
    c = Case(dev, 41, 128, 2, 4, 16, [2, 1], [400, 350], "bf16", window=60)
    y, l = c.run()
    c.check(y, l)
    table = c.table.copy()
    table[0, : (400 - 2 - 60) // 16], table[1, :17] = -1, 2 ** 31 - 1
    y2, l2 = c.run(table=table)
    assert bits((y, y2), (l, l2))


def test_pitches_no_lse_and_no_row_start(dev):
    c = Case(dev, 51, 64, 2, 3, 32, [1, 1, 1], [90, 200, 31], "f16")
    y, l = c.run()
    c.check(y, l)
    y2, l2 = c.run(ld=6 * 64 + 40, lse=False)
    assert bits((y, y2)) and (l2.view(np.uint32) == 0x7E017E01).all()
    y3, l3 = c.run(start=False)
    assert bits((y[:3], y3[:3]), (l[:3], l3[:3]))


def test_bounds_of_the_host_cut(dev):
    """Rows past max_rows stay; tokens past max_length are not there."""
    c = Case(dev, 52, 64, 1, 2, 16, [10, 40], [100, 300], "f16")
    y, l = c.run(max_rows=20)
    assert (y[30:].view(np.uint16) == 0x7E01).all()
    full = c.run()
    c.lengths = np.array([100, 200])
    y, l = c.run(max_length=200)
    c.check(y, l)
    c.lengths = np.array([100, 300])
    y2, l2 = c.run(max_length=200)                                                        # the door cuts 300 to 200
    assert bits((y, y2), (l, l2)) and not bits((full[0], y2))


@pytest.mark.parametrize("bound", [1, 7, 20, 39])
def test_rows_within_the_hosts_bound_keep_their_positions(dev, bound):
    """A sequence of more rows than the host allowed: the ones that are done stand where they stood."""
    c = Case(dev, 53, 64, 1, 2, 16, [10, 40], [100, 300], "bf16")
    y, l = c.run()
    got, lse = c.run(max_rows=bound)
    for s, n in enumerate((10, 40)):
        done, all_ = slice(c.start[s], c.start[s] + min(n, bound)), slice(c.start[s], c.start[s + 1])
        left = slice(done.stop, all_.stop)
        assert (got[left].view(np.uint16) == 0x7E01).all() and (lse[left].view(np.uint32) == 0x7E017E01).all()
        y[done], l[done] = got[done], lse[done]
    c.check(y, l)


@pytest.mark.parametrize("rows,lengths", [([1, 1], [40, 9]), ([1], [3000]), ([30, 2], [300, 17]), ([200], [2000])])
@pytest.mark.parametrize("t", ["f16", "bf16"])
def test_scaled_scores_past_the_range(dev, rows, lengths, t):
    """Every row has a scaled score over fp32's range, some have one below it: NaN, not a row of zeros."""
    c = Case(dev, 54, 64, 2, 3, 32, rows, lengths, t, std=4.0, scale=1.6e38, noise=False)
    y, l = c.run()
    for s, n in enumerate(lengths):
        a, b = c.start[s], c.start[s + 1]
        k, _ = c.cache.tokens(c.table[s], n)
        x = np.einsum("ihd,htd->iht", decode(c.q[a:b], t).astype(np.float64), np.repeat(k, 3, 0))
        for i in range(b - a):
            assert (x[i, :, : n - (b - a) + i + 1].max(axis=1) * 1.6e38 > 1.01 * 2.0 ** 128).all()
        assert np.isnan(decode(y[a:b], t)).all() and np.isnan(l[a:b]).all()


def test_captured_over_a_growing_sequence(dev):
    """A step's graph is captured at the largest length and replayed at all: lengths and rows live on the device."""
    c = Case(dev, 61, 128, 2, 5, 16, [1, 1], [900, 700], "bf16")
    st, heads = qwhip.Stream(dev), 10
    bufs = [dev.put(a) for a in (c.q, c.cache.bytes, c.start, c.lengths.astype(np.int32), c.table)]
    out, le, ws = dev.alloc(c.q.nbytes), dev.alloc(c.total * heads * 4), dev.alloc(1 << 22)
    view = qwhip.KvCache(bufs[1].ptr, c.cache.bytes.nbytes, len(c.cache.bytes), 16, 2, 128)
    batch = qwhip.KvBatch(bufs[2].ptr, bufs[3].ptr, bufs[4].ptr, c.table.shape[1], 2, 1, 900)
    graph = qwhip.Graph(st, lambda: qwhip.check(dev.lib.qwhip_kv_attention_mxfp4(st.handle, C.byref(view), C.byref(batch), bufs[0].ptr, qwhip.BF16, heads, 0, c.total, c.scale, 0, out.ptr,
                                                                                 0, le.ptr, ws.ptr, ws.nbytes)))
    for lengths in ([900, 700], [1, 2], [333, 0], [500, 699], [900, 700]):
        c.lengths = np.array(lengths)
        bufs[3].upload(c.lengths.astype(np.int32))
        qwhip.check(dev.lib.qwhip_fill_u32(st.handle, ws.ptr, 0xFFFFFFFF, ws.nbytes // 4))   # what the workspace held does not matter
        for b in (out, le):
            qwhip.check(dev.lib.qwhip_fill_u32(st.handle, b.ptr, 0x7E017E01, b.nbytes // 4))
        graph.launch()
        st.sync()
        c.check(out.download(np.uint16, c.q.shape), le.download(np.float32, (c.total, heads)))
    graph.destroy()
    for b in (*bufs, out, le, ws):
        b.free()


def test_two_streams_at_once(dev):
    a, b = Case(dev, 71, 128, 2, 4, 64, [1], [3000], "f16"), Case(dev, 72, 128, 2, 4, 64, [1], [3000], "f16")
    want = [a.run(), b.run()]
    other = qwhip.Stream(dev)
    for _ in range(3):
        got = [a.run(stream=other), b.run()]
        for g, w in zip(got, want):
            assert bits((g[0], w[0]), (g[1], w[1]))


def test_pages_past_four_gigabytes(dev):
    """A cache of 5 GB whose last pages are read and written: offsets past 32 bits."""
    page, heads, d = 256, 8, 128
    small = Case(dev, 81, d, heads, 2, page, [3], [700], "bf16")
    piece = dev.lib.qwhip_kv_page_bytes(page, heads, d)
    count = (5 << 30) // piece
    big = dev.alloc(count * piece)
    ids = np.array([[count - 1, count - 3, 11]], np.int32)
    for i, p in enumerate(small.table[0]):
        one = small.cache.bytes[p]
        qwhip.check(dev.lib.qwhip_memcpy_h2d(dev.stream.handle, big.ptr + int(ids[0, i]) * piece, one.ctypes.data, one.nbytes))
    bufs = [dev.put(a) for a in (small.q, small.start, small.lengths.astype(np.int32), ids)]
    out = dev.alloc(small.q.nbytes)
    qwhip.check(dev.lib.qwhip_fill_u32(dev.stream.handle, out.ptr, 0x7E017E01, out.nbytes // 4))
    view, batch = qwhip.KvCache(big.ptr, count * piece, count, page, heads, d), qwhip.KvBatch(bufs[1].ptr, bufs[2].ptr, bufs[3].ptr, 3, 1, 3, 700)
    qwhip.check(dev.lib.qwhip_kv_attention_mxfp4(dev.stream.handle, C.byref(view), C.byref(batch), bufs[0].ptr, qwhip.BF16, 16, 0, small.total, small.scale, 0, out.ptr, 0, None, None, 0))
    dev.stream.sync()
    want, _ = small.run(room=0)
    assert np.array_equal(out.download(np.uint16, small.q.shape), want)
    # and a token appended into the last page
    x = qo.f32_to_bf16_bits(np.random.default_rng(1).standard_normal((1, 2 * heads * d)).astype(np.float32))
    slot = np.array([(count - 1) * page + 9], np.int32)
    xb, sb = dev.put(x), dev.put(slot)
    qwhip.check(dev.lib.qwhip_kv_append_mxfp4(dev.stream.handle, C.byref(view), None, 1, sb.ptr, xb.ptr, 0, xb.ptr + heads * d * 2, 0, qwhip.BF16, None, 0, 0, None, 0, 0, None, None))
    dev.stream.sync()
    got = np.empty((1, heads, piece // heads), np.uint8)
    qwhip.check(dev.lib.qwhip_memcpy_d2h(dev.stream.handle, got.ctypes.data, big.ptr + (count - 1) * piece, piece))
    last = qwkv.Cache(1, page, heads, d)
    last.bytes[0] = small.cache.bytes[small.table[0, 0]]
    val = qo.bf16_bits_to_f32(x).reshape(1, 2 * heads, d)
    last.put(np.array([9]), val[:, :heads], val[:, heads:])
    assert np.array_equal(got, last.bytes)
    for b in (big, *bufs, out, xb, sb):
        b.free()


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("t", ["f16", "bf16"])
def test_many_rows_over_every_page(dev, page, d, t):
    """Tiles in one page and over several, last tiles of every filling, ranges of a window that begin inside a page."""
    c = Case(dev, page + d, d, 2, 3, page, [50, 129, 7, 64], [50, 517, 261, 64 + page // 2 + 3], t)
    c.check(*c.run())
    c.window = 77
    c.check(*c.run())


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("d,rows", [(64, 1), (128, 1), (64, 40), (128, 90), (256, 33)])
def test_a_part_in_the_wide_form_beside_others(dev, d, rows, page, t):
    """Scales past the half types, and a broken block, in one place of a long sequence: the part that meets them covers its own tokens and no others."""
    c = Case(dev, 91 + d, d, 2, 4, page, [rows, 1], [3001, 1500], t, std=0.5)
    kc, ks, vc, vs = c.cache.planes()
    for token, byte in ((1700, 100), (1733, 145 if t == "bf16" else 138), (2990, 255)):
        p, o = c.table[0][token // page], token % page
        vs[p, 0, o // 8, d // 32 - 1, o % 8] = byte
    p, o = c.table[1][640 // page], 640 % page
    ks[p, 1, o] = 96
    y, l = c.run()
    assert c.need > 0 and c.need // (c.total * 8 * (d + 2) * 4) > 1
    c.check(y, l)
    y0, l0 = c.run(room=0)
    c.check(y0, l0)


def test_a_sequence_longer_than_the_parts_there_are(dev):
    c = Case(dev, 95, 64, 1, 2, 64, [2], [70000], "bf16", std=3.0)
    c.check(*c.run())
    assert c.need // (c.total * 2 * 66 * 4) == 256


def test_group_of_one_and_the_largest_group(dev):
    for shared, heads in ((1, 5), (64, 1)):
        c = Case(dev, 96 + shared, 128, heads, shared, 16, [1, 3], [130, 260], "f16")
        c.check(*c.run())
