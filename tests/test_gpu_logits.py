"""qwhip_logits_process through the C ABI against the rules in numpy (oracle/qwmx.py).  Every operation of the rules is one IEEE fp32 operation
in a stated order, so fp32 results are equal bit for bit, 16-bit ones are those results rounded once, and the tokens are equal."""
import ctypes as C

import numpy as np
import pytest

from oracle import qwmx
from oracle import qworacle as qo
from qwegn_amd import qwhip

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return qwhip.Device(0)


def pack_mask(allowed, words):
    out = np.zeros((len(allowed), words), np.uint32)
    for m, row in enumerate(allowed):
        at = np.nonzero(row)[0]
        np.bitwise_or.at(out[m], at >> 5, np.uint32(1) << (at & 31).astype(np.uint32))
    return out


class Step:
    """A batch's rules, on the host and on the device."""

    def __init__(self, dev, rows, n, hist=0, biases=0, masks=0, seed=0, extra_words=0):
        rng = np.random.default_rng(seed)
        self.dev, self.rows, self.n, self.bufs = dev, rows, n, []
        self.host, self.rules = {}, qwhip.LogitsRules()
        h = self.host
        if hist:
            h["hist"] = (rng.random((rows, hist)) ** 3 * n).astype(np.int32)
            h["hist"][rng.random((rows, hist)) < 0.05] = rng.choice([-1, n, n + 7, -2 ** 31, 2 ** 31 - 1])
            h["total"] = rng.integers(0, hist + 1, rows).astype(np.int32)
            h["prompt"] = rng.integers(-2, hist + 3, rows).astype(np.int32)
            h["total"][0] = hist + 5                       # clamped to what is there
            h["rep"], h["pres"], h["freq"] = (1.0 + 0.5 * rng.random(rows)).astype(np.float32), rng.random(rows).astype(np.float32), rng.random(rows).astype(np.float32)
            for field, key in (("history", "hist"), ("total_len", "total"), ("prompt_len", "prompt"), ("repetition", "rep"), ("presence", "pres"), ("frequency", "freq")):
                self.give(field, h[key])
            self.rules.ld_history = hist
        if biases:
            counts = rng.integers(0, biases + 1, rows)
            off = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
            tok = rng.integers(-1, n + 1, off[-1]).astype(np.int32)
            tok[1::3] = tok[0::3][: len(tok[1::3])]        # the same token twice in a row, and across rows
            val = (4 * rng.random(off[-1]) - 2).astype(np.float32)
            h["bias"] = [list(zip(tok[a:b].tolist(), val[a:b].tolist())) for a, b in zip(off[:-1], off[1:])]
            self.give("bias_off", off)
            self.give("bias_tok", tok)
            self.give("bias_val", val)
            self.rules.bias_count = len(tok)
        if masks:
            h["allowed"] = rng.random((masks, n)) < 0.3
            if masks > 1:
                h["allowed"][1] = False
            if masks > 2:
                h["allowed"][2] = False
                h["allowed"][2, n - 1] = True
            h["allowed_row"] = rng.integers(-1, masks + 1, rows).astype(np.int32)
            h["allowed_row"][: min(rows, masks)] = np.arange(min(rows, masks))
            self.rules.ld_allowed = (n + 31) // 32 + extra_words
            self.give("allowed", pack_mask(h["allowed"], self.rules.ld_allowed))
            self.give("allowed_row", h["allowed_row"])
            self.rules.allowed_rows = masks

    def give(self, field, arr):
        b = self.dev.put(arr)
        self.bufs.append(b)
        setattr(self.rules, field, b.ptr)

    def free(self):
        for b in self.bufs:
            b.free()


def image_of(x, t):
    if t == qwhip.BF16:
        b = qo.f32_to_bf16_bits(x.astype(np.float32))
        return b, qo.bf16_bits_to_f32(b)
    a = x.astype(qwhip.NP_DTYPES[t])
    return a, a.astype(np.float32)


def rounded(x, t):
    with np.errstate(over="ignore"):
        return qo.f32_to_bf16_bits(x) if t == qwhip.BF16 else x.astype(qwhip.NP_DTYPES[t])


def run(dev, step, image, t, ld=0, ld_out=0, in_place=False, want_out=True, want_tokens=True, stream=None):
    rows, n = image.shape
    pitch, pitch_out = ld or n, ld_out or n
    wide = np.zeros((rows, pitch), image.dtype)
    wide[:, :n] = image
    src = dev.put(wide)
    size = image.dtype.itemsize
    out = src if in_place else dev.put(np.full(rows * pitch_out * size + 256, 0xA5, np.uint8))
    tok = dev.put(np.full(rows + 4, 77, np.int32))
    room = dev.put(np.full(dev.lib.qwhip_logits_workspace_bytes(rows, n) + 64, 0xFF, np.uint8))
    st = (stream or dev.stream).handle
    qwhip.check(dev.lib.qwhip_logits_process(st, C.byref(step.rules), src.ptr, t, rows, n, ld, out.ptr if want_out else None, ld_out, tok.ptr if want_tokens else None,
                                             room.ptr if want_tokens else None, room.nbytes - 64 if want_tokens else 0))
    dev.stream.sync()
    tokens = tok.download(np.int32, (rows + 4,), stream)
    assert (tokens[rows:] == 77).all()
    got = None
    if in_place:
        got = out.download(image.dtype, (rows, pitch), stream)[:, :n]
    elif want_out:
        raw = out.download(np.uint8, (rows * pitch_out * size + 256,), stream)
        assert (raw[rows * pitch_out * size:] == 0xA5).all()
        body = raw[: rows * pitch_out * size].view(image.dtype).reshape(rows, pitch_out)
        assert (np.ascontiguousarray(body[:, n:]).view(np.uint8) == 0xA5).all()
        got = body[:, :n]
    for b in {id(b): b for b in (src, out, tok, room)}.values():
        b.free()
    return got, tokens[:rows]


def equal(a, b):
    """Bit for bit, but for which NaN a NaN is."""
    fa, fb = (qo.bf16_bits_to_f32(v).astype(np.float32) if v.dtype == np.uint16 else v.astype(np.float32) for v in (a, b))
    nan = np.isnan(fb)
    return np.array_equal(np.isnan(fa), nan) and np.array_equal(np.where(nan, 0, a), np.where(nan, 0, b))


CASES = [dict(rows=1, n=151936, hist=4096, biases=16, masks=1), dict(rows=3, n=1, hist=5, biases=2, masks=2), dict(rows=9, n=32003, hist=257, biases=40, masks=5),
         dict(rows=5, n=2048, hist=1, biases=0, masks=0), dict(rows=17, n=2049, hist=0, biases=300, masks=17), dict(rows=4, n=4097, hist=0, biases=0, masks=3),
         dict(rows=70, n=1003, hist=64, biases=3, masks=20), dict(rows=2, n=8192, hist=20000, biases=0, masks=0), dict(rows=6, n=31, hist=12, biases=4, masks=4),
         dict(rows=130, n=16384, hist=33, biases=2, masks=7), dict(rows=300, n=5000, hist=9, biases=1, masks=3)]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(v) for v in c.values()))
@pytest.mark.parametrize("t", [qwhip.F32, qwhip.F16, qwhip.BF16])
def test_rules(dev, case, t):
    step = Step(dev, seed=case["n"], **case)
    image, val = image_of(np.random.default_rng(case["rows"]).standard_normal((case["rows"], case["n"])) * 3, t)
    want, tokens = qwmx.logits_f32(val, **step.host)
    got, tok = run(dev, step, image, t)
    assert equal(got, rounded(want, t))
    assert np.array_equal(tok, tokens)
    step.free()


def test_nothing_to_apply_is_the_argmax(dev):
    rng = np.random.default_rng(1)
    x = rng.standard_normal((4, 40000)).astype(np.float32)
    x[0, 17] = x[0, 23456] = 50.0                                                      # a tie over two slices: the lower token
    x[1] = -np.inf
    x[2] = np.nan
    x[2, 39999] = -3.0
    x[3] = np.nan
    step = Step(dev, 4, 40000)
    got, tok = run(dev, step, x, qwhip.F32)
    assert equal(got, x)
    assert tok.tolist() == [17, -1, 39999, -1]
    src, out = dev.put(x), dev.alloc(16)
    qwhip.check(dev.lib.qwhip_argmax_f32(dev.stream.handle, src.ptr, 4, 40000, out.ptr))
    dev.stream.sync()
    assert out.download(np.int32, (4,))[[0, 2]].tolist() == [17, 39999]                # the key rule of the fold beside it
    src.free()
    out.free()


def test_infinities_and_nan_under_masks_and_penalties(dev):
    n = 3001
    x = np.random.default_rng(2).standard_normal((6, n)).astype(np.float32)
    x[:, ::7], x[:, 1::7], x[:, 2::7] = np.inf, -np.inf, np.nan
    x[:, 3::7] = np.finfo(np.float32).min
    step = Step(dev, 6, n, hist=200, biases=50, masks=4, seed=3)
    want, tokens = qwmx.logits_f32(x, **step.host)
    got, tok = run(dev, step, x, qwhip.F32)
    assert equal(got, want)
    assert np.array_equal(tok, tokens)
    step.free()


@pytest.mark.parametrize("t", [qwhip.F32, qwhip.BF16])
@pytest.mark.parametrize("ld,ld_out,in_place", [(5003, 5011, False), (5001, 5001, True), (5008, 0, False), (0, 0, True), (5004, 5001, False)])
def test_pitches_and_in_place(dev, t, ld, ld_out, in_place):
    rows, n = 7, 5000
    step = Step(dev, rows, n, hist=100, biases=5, masks=3, extra_words=3)
    image, val = image_of(np.random.default_rng(4).standard_normal((rows, n)), t)
    want, tokens = qwmx.logits_f32(val, **step.host)
    got, tok = run(dev, step, image, t, ld=ld, ld_out=ld_out, in_place=in_place)
    assert equal(got, rounded(want, t))
    assert np.array_equal(tok, tokens)
    step.free()


def test_tokens_alone_and_logits_alone(dev):
    rows, n = 5, 9000
    step = Step(dev, rows, n, hist=300, biases=9, masks=5)
    x = np.random.default_rng(5).standard_normal((rows, n)).astype(np.float32)
    want, tokens = qwmx.logits_f32(x, **step.host)
    _, tok = run(dev, step, x, qwhip.F32, want_out=False)
    assert np.array_equal(tok, tokens)
    got, untouched = run(dev, step, x, qwhip.F32, want_tokens=False)
    assert equal(got, want)
    assert (untouched == 77).all()
    step.free()


def test_bias_offsets_outside_the_list_are_clamped(dev):
    step = Step(dev, 3, 100)
    step.give("bias_off", np.array([-5, 2, 1, 900], np.int32))
    step.give("bias_tok", np.array([3, 4, 5, 5], np.int32))
    step.give("bias_val", np.array([1, 2, 3, 4], np.float32))
    step.rules.bias_count = 4
    x = np.zeros((3, 100), np.float32)
    got, tok = run(dev, step, x, qwhip.F32)
    want = np.zeros((3, 100), np.float32)
    want[0, 3], want[0, 4], want[2, 4], want[2, 5] = 1, 2, 2, 4
    assert np.array_equal(got, want)
    assert tok.tolist() == [4, 0, 5]
    step.free()


def test_captured_beside_another_stream(dev):
    rows, n = 3, 20000
    step = Step(dev, rows, n, hist=500, biases=4, masks=2)
    x = np.random.default_rng(6).standard_normal((rows, n)).astype(np.float32)
    want, tokens = qwmx.logits_f32(x, **step.host)
    src, graphs = dev.put(x), []
    for _ in range(2):
        st = qwhip.Stream(dev)
        out, tok, room = dev.alloc(rows * n * 4), dev.alloc(64), dev.alloc(dev.lib.qwhip_logits_workspace_bytes(rows, n))
        call = lambda st=st, out=out, tok=tok, room=room: qwhip.check(dev.lib.qwhip_logits_process(  # noqa: E731
            st.handle, C.byref(step.rules), src.ptr, qwhip.F32, rows, n, 0, out.ptr, 0, tok.ptr, room.ptr, room.nbytes))
        graphs.append((qwhip.Graph(st, call), st, out, tok, room))
    for _ in range(3):
        for _, _, out, tok, _ in graphs:
            qwhip.check(dev.lib.qwhip_fill_u32(dev.stream.handle, out.ptr, 0, rows * n))
            qwhip.check(dev.lib.qwhip_fill_u32(dev.stream.handle, tok.ptr, 0, rows))
        dev.stream.sync()
        for g, *_ in graphs:
            g.launch()
        for _, st, out, tok, _ in graphs:
            st.sync()
            assert equal(out.download(np.float32, (rows, n)), want)
            assert np.array_equal(tok.download(np.int32, (rows,)), tokens)
    for g, _, *bufs in graphs:
        g.destroy()
        for b in bufs:
            b.free()
    src.free()
    step.free()
