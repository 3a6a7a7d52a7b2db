"""qwhip_logits_process where a row's slices, ties and zeros can go wrong, against the rules in numpy (oracle/qwmx.py), bit for bit."""
import ctypes as C

import numpy as np
import pytest

from oracle import qwmx
from oracle import qworacle as qo
from qwegn_amd import qwhip
from tests.test_gpu_logits import Step, equal, image_of, rounded, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return qwhip.Device(0)


@pytest.mark.parametrize("t", [qwhip.F32, qwhip.F16, qwhip.BF16])
@pytest.mark.parametrize("rows,n", [(3, 9), (1, 40000), (130, 16384), (256, 32003)])
def test_zeros_of_both_signs(dev, t, rows, n):
    """A row whose largest result is a zero: +0 is above -0, as the fold of qwhip_argmax_f32 has it, then the lower token wins."""
    rng = np.random.default_rng(n)
    x = -np.abs(rng.standard_normal((rows, n))) - 0.01
    for r in range(rows):
        low, high = np.sort(rng.choice(n, 2, replace=False))
        x[r, low], x[r, high] = ((-0.0, 0.0), (0.0, -0.0), (-0.0, -0.0), (0.0, 0.0))[r % 4]
    if n > 2048:
        x[rows - 1] = -1.0
        x[rows - 1, [7, 7 + 1024, 9]] = -0.0, 0.0, -0.0      # one thread's own where it has several
    image, val = image_of(x, t)
    assert (np.signbit(val) | (val == 0)).all()
    step = Step(dev, rows, n)
    want, tokens = qwmx.logits_f32(val)
    assert np.array_equal(tokens, qo.head_argmax(val))
    got, tok = run(dev, step, image, t)
    assert equal(got, rounded(want, t))
    assert np.array_equal(tok, tokens)
    src, out = dev.put(val), dev.alloc(rows * 4)
    qwhip.check(dev.lib.qwhip_argmax_f32(dev.stream.handle, src.ptr, rows, n, out.ptr))
    dev.stream.sync()
    assert np.array_equal(out.download(np.int32, (rows,)), tokens)
    src.free()
    out.free()


def tokens_a_thread(rows, n):
    """The launch's rule: the most of 16, 8, 4, 2, 1 that leave 512 workgroups."""
    each = 16
    while each > 1 and rows * -(-n // (1024 * each)) < 512:
        each //= 2
    return each


FORMS = [(16, dict(rows=520, n=1003, hist=40, biases=5, masks=7)), (16, dict(rows=260, n=16390, hist=700, biases=20, masks=3)), (16, dict(rows=256, n=32003, hist=33, biases=3, masks=0)),
         (16, dict(rows=256, n=16385, hist=0, biases=9, masks=256)), (8, dict(rows=256, n=8193, hist=1500, biases=4, masks=5)), (8, dict(rows=130, n=32003, hist=129, biases=30, masks=40)),
         (16, dict(rows=512, n=8192, hist=5, biases=0, masks=0)), (4, dict(rows=130, n=16384, hist=260, biases=2, masks=4)), (4, dict(rows=171, n=8195, hist=70, biases=7, masks=9)),
         (2, dict(rows=130, n=8000, hist=100, biases=6, masks=6)), (2, dict(rows=130, n=6145, hist=2000, biases=0, masks=3)), (1, dict(rows=20, n=25601, hist=300, biases=8, masks=2))]


@pytest.mark.parametrize("each,case", FORMS, ids=lambda c: "-".join(str(v) for v in c.values()) if isinstance(c, dict) else f"e{c}")
@pytest.mark.parametrize("t", [qwhip.F32, qwhip.F16, qwhip.BF16])
def test_every_number_of_tokens_a_thread(dev, t, each, case):
    """Slices that end with one token, with part of a thread's and whole; logits on a coarse grid, so that a row's largest stands in several
    threads and slices."""
    rows, n = case["rows"], case["n"]
    assert tokens_a_thread(rows, n) == each
    step = Step(dev, seed=n, **case)
    rng = np.random.default_rng(rows + n)
    x = rng.integers(-12, 13, (rows, n)) / 4.0
    x[np.arange(rows), rng.integers(0, n, rows)] = 3.25     # a single largest in some rows, beaten by rules or masks in others
    x[: rows // 2, -1] = 3.25                               # the last slice's last token
    x[::3] = np.minimum(x[::3], 3.0)                        # ties of many
    image, val = image_of(x, t)
    want, tokens = qwmx.logits_f32(val, **step.host)
    got, tok = run(dev, step, image, t)
    assert equal(got, rounded(want, t))
    assert np.array_equal(tok, tokens)
    step.free()


@pytest.mark.parametrize("t", [qwhip.F32, qwhip.BF16])
@pytest.mark.parametrize("each,rows,n,ld", [(16, 256, 16385, 16400), (8, 256, 8193, 0), (2, 130, 6145, 6147)])
def test_wide_slices_in_place_and_with_odd_values(dev, t, each, rows, n, ld):
    assert tokens_a_thread(rows, n) == each
    step = Step(dev, rows, n, hist=200, biases=12, masks=6, seed=9, extra_words=2)
    x = np.random.default_rng(7).standard_normal((rows, n)).astype(np.float32)
    x[:, ::7], x[:, 1::7], x[:, 2::7], x[:, 3::7] = np.inf, -np.inf, np.nan, -3.0e38
    x[1::2, ::7] = 0.0
    image, val = image_of(x, t)
    want, tokens = qwmx.logits_f32(val, **step.host)
    got, tok = run(dev, step, image, t, ld=ld, ld_out=ld, in_place=True)
    assert equal(got, rounded(want, t))
    assert np.array_equal(tok, tokens)
    _, alone = run(dev, step, image, t, ld=ld, want_out=False)
    assert np.array_equal(alone, tokens)
    step.free()


def test_wide_slices_captured(dev):
    """A full batch's form, recorded: histories grow between the replays."""
    rows, n, room_for = 256, 16385, 64
    rng = np.random.default_rng(8)
    x = rng.standard_normal((rows, n)).astype(np.float32)
    hist, lens = rng.integers(0, n, (rows, room_for)).astype(np.int32), np.zeros(rows, np.int32)
    freq = np.full(rows, 0.5, np.float32)
    src, hb, lb, fb = dev.put(x), dev.put(hist), dev.put(lens), dev.put(freq)
    out, tok, room = dev.alloc(rows * n * 4), dev.alloc(rows * 4), dev.alloc(dev.lib.qwhip_logits_workspace_bytes(rows, n))
    rules = qwhip.LogitsRules(history=hb.ptr, total_len=lb.ptr, frequency=fb.ptr, ld_history=room_for)
    st = qwhip.Stream(dev)
    g = qwhip.Graph(st, lambda: qwhip.check(dev.lib.qwhip_logits_process(st.handle, C.byref(rules), src.ptr, qwhip.F32, rows, n, 0, out.ptr, 0, tok.ptr, room.ptr,
                                                                        room.nbytes)))
    for turn in range(4):
        qwhip.check(dev.lib.qwhip_fill_u32(dev.stream.handle, out.ptr, 0, rows * n))
        qwhip.check(dev.lib.qwhip_fill_u32(dev.stream.handle, room.ptr, 0xFFFFFFFF, room.nbytes // 4))
        dev.stream.sync()
        g.launch()
        st.sync()
        want, tokens = qwmx.logits_f32(x, hist=hist, total=lens, freq=freq)
        assert np.array_equal(out.download(np.float32, (rows, n)), want), turn
        assert np.array_equal(tok.download(np.int32, (rows,)), tokens)
        for r in range(rows):
            hist[r, lens[r]] = tokens[r]
        lens += 1 + np.arange(rows, dtype=np.int32) % 7
        hb.upload(hist)
        lb.upload(lens)
    g.destroy()
    for b in (src, hb, lb, fb, out, tok, room):
        b.free()
