"""qwhip_kv_attention_mxfp4 and memory that a row does not see: what stands in front of a window or behind the last row of a workgroup's tile, in pages that belong to someone
else by now or in the sequence's own, changes no bit."""
import numpy as np
import pytest

from qwegn_amd import qwhip
from tests.test_gpu_attention import Case, bits
from tests.test_gpu_attention_tiles import Tiles

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return qwhip.Device(0)


def spoil(c, pages, seed=9):
    """Codes of noise and scale bytes past both half types' range (broken blocks among them) in these pages."""
    rng = np.random.default_rng(seed)
    kc, ks, vc, vs = c.cache.planes()
    for p in pages:
        c.cache.bytes[p] = rng.integers(0, 256, c.cache.bytes[p].shape)
        ks[p], vs[p] = rng.choice([1, 99, 230, 253, 255], ks[p].shape), rng.choice([1, 99, 230, 253, 255], vs[p].shape)


def without_page_zero(c):
    """Page 0, as which an entry outside of the cache is read, in no table."""
    other = (set(range(1, len(c.cache.bytes))) - set(c.table[:, : c.each].reshape(-1).tolist())).pop()
    at = c.table[:, : c.each] == 0
    if at.any():
        c.cache.bytes[other] = c.cache.bytes[0]
        c.table[:, : c.each][at] = other


# a window is the bound of a sequence's tokens: many heads and rows make up for it where the tile kernel is to be called for
WINDOWS = [(Case, d, page, 2, 4, [2, 1, 1, 30], [400, 350, 95, 333], w) for d in (64, 128, 256) for page in (16, 32, 64) for w in (1, 17, 60)] + \
          [(Tiles, d, page, 32, 16, [300, 300, 300], [340, 473, 395], w) for d in (64, 128) for page in (16, 32, 64, 128) for w in (1, 60)]


@pytest.mark.parametrize("cls,d,page,heads,shared,rows,lengths,window", WINDOWS)
@pytest.mark.parametrize("t", ["f16", "bf16"])
def test_pages_in_front_of_a_window(dev, cls, d, page, heads, shared, rows, lengths, window, t):
    """Freed pages: entries outside of the cache over a page 0 that is not the sequences', entries of pages that another sequence has filled since.  Bits as before."""
    c = cls(dev, d + page + window, d, heads, shared, page, rows, lengths, t, window=window)
    without_page_zero(c)
    y, l = c.run(room=1 << 26)
    if cls is Case:
        c.check(y, l)
    table, gone = c.table.copy(), []
    for s, (n, length) in enumerate(zip(rows, lengths)):
        first = max(0, length - n - window + 1) // page                                   # the page of the first token that the first row sees
        gone += table[s, :first].tolist()
        table[s, :first] = -1
    spoil(c, [0])
    got = c.run(room=1 << 26, table=table)
    assert bits((y, got[0]), (l, got[1]))
    spoil(c, gone)
    got = c.run(room=1 << 26)
    assert bits((y, got[0]), (l, got[1]))


@pytest.mark.parametrize("cls,d,page,rows,lengths", [(Case, 64, 16, [1, 2], [400, 350]), (Case, 128, 64, [1, 2], [401, 350]), (Case, 256, 32, [3, 1], [250, 77]), (Tiles, 64, 128, [600], [663]),
                                                      (Tiles, 128, 64, [600], [663])])
@pytest.mark.parametrize("t", ["f16", "bf16"])
def test_tokens_in_front_of_a_window_in_its_first_page(dev, cls, d, page, rows, lengths, t):
    """Blocks out of the half types' range, or broken, in the page that a window begins in, in front of it."""
    c = cls(dev, d + page, d, *((2, 4) if cls is Case else (32, 16)), page, rows, lengths, t)
    for window in (45, 58):
        c.window = window
        y, l = c.run(room=1 << 26)
        kept = c.cache.bytes.copy()
        kc, ks, vc, vs = c.cache.planes()
        for s, (n, length) in enumerate(zip(rows, lengths)):
            for token in range(max(0, length - n - window + 1)):
                p, o = c.table[s][token // page], token % page
                ks[p, :, o], vs[p, :, o // 8, :, o % 8] = (230, 255)[token % 2], (255, 99)[token % 2]
        got = c.run(room=1 << 26)
        c.cache.bytes[:] = kept
        assert bits((y, got[0]), (l, got[1])), window


@pytest.mark.parametrize("cls,d,page,rows", [(Case, 64, 16, 30), (Case, 128, 64, 30), (Case, 256, 32, 20), (Tiles, 64, 16, 130), (Tiles, 64, 128, 130), (Tiles, 128, 64, 130)])
@pytest.mark.parametrize("t", ["f16", "bf16"])
def test_tokens_behind_a_tiles_last_row(dev, cls, d, page, rows, t):
    """The last tokens of a prompt broken or out of range: the rows whose tiles end in front of them keep their bits."""
    c = cls(dev, d + rows, d, 2, 4, page, [rows], [rows], t)
    y, l = c.run(room=0)
    kc, ks, vc, vs = c.cache.planes()
    columns = 16 if cls is Case else 128
    for tile in range(1, rows * 4 // columns):
        first = tile * columns // 4                                                       # the tile's first row, and its position
        kept = c.cache.bytes.copy()
        for token in range(first, rows):
            p, o = c.table[0][token // page], token % page
            ks[p, :, o], vs[p, :, o // 8, :, o % 8] = (230, 255)[token % 2], (255, 99)[token % 2]
        got = c.run(room=0)
        c.cache.bytes[:] = kept
        assert bits((y[:first], got[0][:first]), (l[:first], got[1][:first])), tile
