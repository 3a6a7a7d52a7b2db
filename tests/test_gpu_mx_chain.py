"""The MXFP4 doors and the logits' rules as a serving program strings them together, on the library's own norm and head argmax: weights
quantised at load, a prompt's rows normed, quantised and multiplied, the last rows' logits from an MXFP4 head, the rules, the tokens; then a
captured decode step that is replayed while the requests' histories grow."""
import ctypes as C

import numpy as np
import pytest

from oracle import qwmx
from qwegn_amd import qwhip
from tests.test_gpu_logits import pack_mask
from tests.test_gpu_mxfp4 import check_product, free, view

pytestmark = pytest.mark.gpu

HIDDEN, INNER, VOCAB = 512, 1056, 5003


@pytest.fixture(scope="module")
def dev():
    return qwhip.Device(0)


class Model:
    """Two quantised matrices and their values."""

    def __init__(self, dev):
        self.dev, self.bufs = dev, []
        rng = np.random.default_rng(11)
        self.up, self.up_w = self.load(rng.standard_normal((INNER, HIDDEN)).astype(np.float32) * 0.05)
        self.head, self.head_w = self.load(rng.standard_normal((VOCAB, INNER)).astype(np.float32) * 0.05)
        self.gamma = dev.put((rng.standard_normal(HIDDEN) * 0.1).astype(np.float16))

    def load(self, w):
        n, k = w.shape
        src, codes, scales = self.dev.put(w), self.dev.alloc(n * k // 2), self.dev.alloc(n * k // 32)
        qwhip.check(self.dev.lib.qwhip_quantize_mxfp4(self.dev.stream.handle, src.ptr, qwhip.F32, n, k, 0, codes.ptr, scales.ptr, None))
        self.dev.stream.sync()
        src.free()
        self.bufs += [codes, scales]
        c, s = qwmx.quantise(w)
        assert np.array_equal(codes.download(np.uint8, c.shape), c) and np.array_equal(scales.download(np.uint8, s.shape), s)
        return view(codes, scales, n, k), qwmx.values(c, s)


@pytest.fixture(scope="module")
def model(dev):
    return Model(dev)


def test_prompt_and_first_tokens(dev, model):
    rows, last = 150, 7
    rng = np.random.default_rng(12)
    lib, st = dev.lib, dev.stream.handle
    x = rng.standard_normal((rows, HIDDEN)).astype(np.float16)
    xb, normed = dev.put(x), dev.alloc(rows * HIDDEN * 2)
    codes, scales, values = dev.alloc(rows * HIDDEN // 2), dev.alloc(rows * HIDDEN // 32), dev.alloc(rows * HIDDEN * 2)
    inner, logits, out = dev.alloc(rows * INNER * 2), dev.alloc(last * VOCAB * 4), dev.alloc(last * VOCAB * 4)
    tokens, room = dev.alloc(64), dev.alloc(lib.qwhip_logits_workspace_bytes(last, VOCAB))
    need = lib.qwhip_mxfp4_gemm_workspace_bytes(rows, INNER, HIDDEN)
    planes = dev.alloc(need)
    hist = rng.integers(0, VOCAB, (last, 64)).astype(np.int32)
    lens = rng.integers(1, 65, last).astype(np.int32)
    allowed = rng.random((2, VOCAB)) < 0.2
    which = np.array([0, -1, 1, -1, 0, 1, -1], np.int32)
    keep = [dev.put(a) for a in (hist, lens, np.full(last, 1.2, np.float32), pack_mask(allowed, (VOCAB + 31) // 32), which)]
    rules = qwhip.LogitsRules(history=keep[0].ptr, total_len=keep[1].ptr, prompt_len=keep[1].ptr, repetition=keep[2].ptr, allowed=keep[3].ptr, allowed_row=keep[4].ptr,
                              ld_history=64, allowed_rows=2, ld_allowed=(VOCAB + 31) // 32)
    qwhip.check(lib.qwhip_rmsnorm(st, xb.ptr, model.gamma.ptr, None, rows, HIDDEN, 1e-6, 0, normed.ptr))
    qwhip.check(lib.qwhip_quantize_mxfp4(st, normed.ptr, qwhip.F16, rows, HIDDEN, 0, codes.ptr, scales.ptr, values.ptr))
    xv = view(codes, scales, rows, HIDDEN)
    qwhip.check(lib.qwhip_mxfp4_gemm(st, C.byref(model.up), C.byref(xv), inner.ptr, qwhip.F16, 0, planes.ptr, planes.nbytes))
    tail = inner.ptr + (rows - last) * INNER * 2
    qwhip.check(lib.qwhip_mxfp4_gemv(st, C.byref(model.head), tail, qwhip.F16, last, None, logits.ptr))
    qwhip.check(lib.qwhip_logits_process(st, C.byref(rules), logits.ptr, qwhip.F32, last, VOCAB, 0, out.ptr, 0, tokens.ptr, room.ptr, room.nbytes))
    dev.stream.sync()
    # every step against its definition on what the step before it left
    n16 = normed.download(np.float16, (rows, HIDDEN))
    c, s = qwmx.quantise(n16)
    assert np.array_equal(codes.download(np.uint8, c.shape), c) and np.array_equal(scales.download(np.uint8, s.shape), s)
    xq = qwmx.values(c, s)
    assert np.array_equal(values.download(np.float16, xq.shape).astype(np.float64), xq)
    i16 = inner.download(np.float16, (rows, INNER))
    check_product(i16.astype(np.float32), xq, model.up_w, qwhip.F16)
    l32 = logits.download(np.float32, (last, VOCAB))
    check_product(l32, i16[rows - last:].astype(np.float64), model.head_w, qwhip.F32)
    want, tok = qwmx.logits_f32(l32, hist=hist, total=lens, prompt=lens, rep=np.full(last, 1.2, np.float32), allowed=allowed, allowed_row=which)
    assert np.array_equal(out.download(np.float32, (last, VOCAB)), want)
    assert np.array_equal(tokens.download(np.int32, (last,)), tok)
    # the plain head fold agrees where no rule applies
    plain = qwhip.LogitsRules()
    qwhip.check(lib.qwhip_logits_process(st, C.byref(plain), logits.ptr, qwhip.F32, last, VOCAB, 0, None, 0, tokens.ptr, room.ptr, room.nbytes))
    dev.stream.sync()
    a = tokens.download(np.int32, (last,))
    qwhip.check(lib.qwhip_argmax_f32(st, logits.ptr, last, VOCAB, tokens.ptr))
    dev.stream.sync()
    assert np.array_equal(a, tokens.download(np.int32, (last,)))
    free(xb, normed, codes, scales, values, inner, logits, out, tokens, room, planes, *keep)


def test_captured_decode_step_with_growing_histories(dev, model):
    rows, room_for = 3, 16
    rng = np.random.default_rng(13)
    lib, st = dev.lib, qwhip.Stream(dev)
    xb, logits, tokens = dev.alloc(rows * INNER * 2), dev.alloc(rows * VOCAB * 4), dev.alloc(64)
    room = dev.alloc(lib.qwhip_logits_workspace_bytes(rows, VOCAB))
    hist, lens = np.full((rows, room_for), -1, np.int32), np.zeros(rows, np.int32)
    hb, lb = dev.put(hist), dev.put(lens)
    freq, pres = np.full(rows, 5.0, np.float32), np.full(rows, 3.0, np.float32)
    fb, pb = dev.put(freq), dev.put(pres)
    rules = qwhip.LogitsRules(history=hb.ptr, total_len=lb.ptr, frequency=fb.ptr, presence=pb.ptr, ld_history=room_for)

    def step():
        qwhip.check(lib.qwhip_mxfp4_gemv(st.handle, C.byref(model.head), xb.ptr, qwhip.BF16, rows, None, logits.ptr))
        qwhip.check(lib.qwhip_logits_process(st.handle, C.byref(rules), logits.ptr, qwhip.F32, rows, VOCAB, 0, logits.ptr, 0, tokens.ptr, room.ptr, room.nbytes))

    x = (rng.standard_normal((rows, INNER)) * 0.5).astype(np.float32)
    image = (x.view(np.uint32) >> 16).astype(np.uint16)                     # truncated to bf16: any numbers do
    val = (image.astype(np.uint32) << 16).view(np.float32)
    xb.upload(image)
    raw = dev.alloc(rows * VOCAB * 4)
    qwhip.check(lib.qwhip_mxfp4_gemv(dev.stream.handle, C.byref(model.head), xb.ptr, qwhip.BF16, rows, None, raw.ptr))
    plain = raw.download(np.float32, (rows, VOCAB))
    check_product(plain, val.astype(np.float64), model.head_w, qwhip.F32)
    g = qwhip.Graph(st, step)
    for turn in range(room_for):
        g.launch()
        st.sync()
        want, tok = qwmx.logits_f32(plain, hist=hist, total=lens, freq=freq, pres=pres)
        got = tokens.download(np.int32, (rows,))
        assert np.array_equal(logits.download(np.float32, (rows, VOCAB)), want), turn
        assert np.array_equal(got, tok)
        hist[:, turn] = got
        lens[:] = turn + 1
        hb.upload(hist)
        lb.upload(lens)
    assert all(len(set(r)) > 3 for r in hist.tolist())                      # the penalties moved the choice
    g.destroy()
    free(xb, logits, tokens, room, hb, lb, fb, pb, raw)
