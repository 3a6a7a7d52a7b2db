"""qwhip_kv_attention_mxfp4 where the host's bounds call for the tile kernel: 256 columns and more (query rows of a group of heads) over at least 2^20 tokens of all
tiles.  The tables here are long enough for a bound of 2^20, so that short sequences go through it too; definition, bounds of the error and noise as beside."""
import ctypes as C

import numpy as np
import pytest

from oracle import qwkv
from qwegn_amd import qwhip
from tests.test_gpu_attention import Case, bits
from tests.test_gpu_heads import decode, encode

pytestmark = pytest.mark.gpu
BOUND = 1 << 20


@pytest.fixture(scope="module")
def dev():
    return qwhip.Device(0)


class Tiles(Case):
    """A case whose bound is 2^20 tokens; what the table holds behind a sequence is noise."""

    def __init__(self, *args, **kw):
        super().__init__(*args, **kw)
        noise = np.random.default_rng(5).integers(-2 ** 31, 2 ** 31, (self.seqs, BOUND // self.page)).astype(np.int32)
        noise[:, : self.each] = self.table
        self.table = noise
        assert max(self.rows) * self.shared >= 256

    def run(self, max_length=None, **kw):
        return super().run(max_length=BOUND if max_length is None else max_length, **kw)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("t", ["f16", "bf16"])
def test_every_page(dev, page, d, t):
    """Tiles in one page and over several, last tiles of every filling, in one part and in many."""
    c = Tiles(dev, page + d, d, 2, 3, page, [50, 129, 7, 64], [50, 517, 261, 64 + page // 2 + 3], t)
    y, l = c.run()
    c.check(y, l)
    tiles = min(4 * 4, c.total * 3 // 128 + 4) * 2
    assert c.need // (c.total * 6 * (d + 2) * 4) == (512 if d == 128 else 768) // tiles
    y0, l0 = c.run(room=0)
    c.check(y0, l0)
    y1, l1 = c.run()
    assert bits((y, y1), (l, l1))


@pytest.mark.parametrize("d,t", [(64, "f16"), (128, "bf16")])
def test_ragged_rows(dev, d, t):
    """Prompts from their first token, chunks behind cached tokens, no rows, no tokens, one row, more rows than tokens (rows that see nothing)."""
    c = Tiles(dev, d, d, 2, 3, 32, [70, 1, 0, 16, 45, 9, 200, 3], [70, 200, 50, 321, 45, 4, 777, 0], t)
    y, l = c.run()
    c.check(y, l)
    for empty in (slice(c.start[5], c.start[5] + 5), slice(c.start[7], c.start[8])):
        assert (decode(y[empty], t) == 0).all() and (l[empty] == -np.inf).all()


@pytest.mark.parametrize("rows,shared", [(16, 16), (256, 1), (64, 4), (300, 1), (512, 1), (27, 23)])
def test_columns_at_the_borders_of_tiles(dev, rows, shared):
    c = Tiles(dev, rows, 64, 1, shared, 64, [rows, 1], [rows + 131, 700], "bf16")
    c.check(*c.run())
    c.check(*c.run(room=0))


@pytest.mark.parametrize("d,t,page", [(64, "bf16", 32), (128, "f16", 64)])
def test_window(dev, d, t, page):
    """A window is the bound then: many heads make up for it.  Some rows of all are looked at."""
    c = Tiles(dev, 7 * d, d, 64, 4, page, [66, 70], [4200, 900], t, window=4000)
    y, l = c.run(room=1 << 26)
    q = decode(c.q, t).astype(np.float64)
    for s, n in enumerate((4200, 900)):
        k, v = c.cache.tokens(c.table[s], n)
        for r in (0, 1, 31, int(c.rows[s]) - 1):
            at, seen = c.start[s] + r, n - int(c.rows[s]) + r + 1
            want, lse, size = qwkv.attention(q[at:at + 1], k[:, :seen], v[:, :seen], float(c.scale), 4000)
            kk = np.repeat(np.abs(k[:, :seen]), 4, 0)
            reach = np.max(np.matmul(kk, np.abs(q[at])[:, :, None])[..., 0], axis=1) * float(c.scale)
            e = (d + 8) * 2.0 ** -24 * reach + 2.0 ** -20
            tol = (2.0 ** -11 if t == "f16" else 2.0 ** -8) * np.abs(want) + (2.0 ** -11 * 1.01 + 2 * e[..., None]) * size + n * 2.0 ** -25 * np.abs(v).max() + 2.0 ** -25
            assert (np.abs(decode(y[at:at + 1], t) - want) <= tol).all(), (s, r)
            assert (np.abs(l[at] - lse[0]) <= e + 2.0 ** -22 * (np.abs(lse[0]) + np.log(n + 2.0))).all(), (s, r)


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
def test_scales_outside_of_the_half_types(dev, d, t):
    """Keys and values far above and below f16's range among ordinary ones, blocks of zeros: every tile goes the wide way."""
    c = Tiles(dev, 22, d, 2, 4, 16, [1, 80, 5], [200, 333, 64], t, std=0.3)
    kc, ks, vc, vs = c.cache.planes()
    rng = np.random.default_rng(4)
    ks[rng.random(ks.shape) < 0.02] = 100
    vs[rng.random(vs.shape) < 0.02] = 100
    vs[rng.random(vs.shape) < 0.01] = 137 if t == "f16" else 150
    ks[rng.random(ks.shape) < 0.01] = 0
    vs[rng.random(vs.shape) < 0.01] = 1
    c.check(*c.run())
    c.check(*c.run(room=0))


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("d", [64, 128])
def test_a_part_in_the_wide_form_beside_others(dev, d, page, t):
    """Scales past the half types, and broken blocks, in few places of long sequences: the parts that meet them cover their own tokens and no others, and
    only the rows and heads that see a broken block get NaN."""
    c = Tiles(dev, 92 + d, d, 2, 4, page, [90, 1], [3001, 1500], t, std=0.5)
    kc, ks, vc, vs = c.cache.planes()
    for token, byte in ((1700, 100), (1733, 145 if t == "bf16" else 138), (2990, 255)):
        p, o = c.table[0][token // page], token % page
        vs[p, 0, o // 8, d // 32 - 1, o % 8] = byte
    p, o = c.table[0][2950 // page], 2950 % page
    ks[p, 1, o, 0] = 255
    p, o = c.table[1][640 // page], 640 % page
    ks[p, 1, o] = 96
    y, l = c.run()
    c.check(y, l)
    got = decode(y, t)
    assert np.isnan(got[79:90, :4, d - 32:]).all() and np.isfinite(got[:79, :4]).all() and np.isnan(got[39:90, 4:]).all() and np.isfinite(got[:39, 4:]).all()
    c.check(*c.run(room=0))


def test_nan_and_infinities_of_a_query_stay_in_its_row_and_head(dev):
    c = Tiles(dev, 35, 128, 2, 3, 16, [90, 1], [150, 200], "bf16")
    x = decode(c.q, "bf16").astype(np.float32)
    x[1, 2, 7], x[77, 0, 1] = np.nan, np.nan
    c.q = encode(x, "bf16")
    c.check(*c.run())


def test_scaled_scores_past_the_range(dev):
    c = Tiles(dev, 55, 64, 2, 4, 32, [80], [2000], "bf16", std=4.0, scale=1.6e38, noise=False)
    for room in (0, 1 << 24):
        y, l = c.run(room=room)
        assert np.isnan(decode(y[:80], "bf16")).all() and np.isnan(l[:80]).all()


@pytest.mark.parametrize("bound", [90, 130])
def test_rows_within_the_hosts_bound_keep_their_positions(dev, bound):
    c = Tiles(dev, 56, 64, 1, 3, 16, [10, 140], [100, 300], "f16")
    y, l = c.run()
    got, lse = c.run(max_rows=bound)
    left = slice(10 + bound, 150)
    assert (got[left].view(np.uint16) == 0x7E01).all() and (lse[left].view(np.uint32) == 0x7E017E01).all()
    y[: 10 + bound], l[: 10 + bound] = got[: 10 + bound], lse[: 10 + bound]
    c.check(y, l)


def test_captured_over_growing_sequences(dev):
    c = Tiles(dev, 62, 128, 2, 4, 64, [70, 30], [900, 700], "bf16")
    st, heads = qwhip.Stream(dev), 8
    bufs = [dev.put(a) for a in (c.q, c.cache.bytes, c.start, c.lengths.astype(np.int32), c.table)]
    out, le, ws = dev.alloc(c.q.nbytes), dev.alloc(c.total * heads * 4), dev.alloc(1 << 24)
    view = qwhip.KvCache(bufs[1].ptr, c.cache.bytes.nbytes, len(c.cache.bytes), 64, 2, 128)
    batch = qwhip.KvBatch(bufs[2].ptr, bufs[3].ptr, bufs[4].ptr, c.table.shape[1], 2, 70, BOUND)
    graph = qwhip.Graph(st, lambda: qwhip.check(dev.lib.qwhip_kv_attention_mxfp4(st.handle, C.byref(view), C.byref(batch), bufs[0].ptr, qwhip.BF16, heads, 0, c.total, c.scale, 0, out.ptr,
                                                                                 0, le.ptr, ws.ptr, ws.nbytes)))
    for lengths in ([900, 700], [70, 2], [333, 0], [500, 699], [900, 700]):
        c.lengths = np.array(lengths)
        bufs[3].upload(c.lengths.astype(np.int32))
        qwhip.check(dev.lib.qwhip_fill_u32(st.handle, ws.ptr, 0xFFFFFFFF, ws.nbytes // 4))
        for b in (out, le):
            qwhip.check(dev.lib.qwhip_fill_u32(st.handle, b.ptr, 0x7E017E01, b.nbytes // 4))
        graph.launch()
        st.sync()
        c.check(out.download(np.uint16, c.q.shape), le.download(np.float32, (c.total, heads)))
    graph.destroy()
    for b in (*bufs, out, le, ws):
        b.free()
