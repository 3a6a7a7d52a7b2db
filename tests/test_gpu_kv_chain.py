"""A layer's attention as a serving program strings it together: norm, the q|k|v projection over a quantised bank, head norms with rotation into the paged
4-bit cache, attention, the output projection whose rotated bank takes the attention's rows as they are; a prompt through the GEMMs, then a captured
decode step of two requests that is replayed while they grow."""
import ctypes as C

import numpy as np
import pytest

from oracle import qwkv
from oracle import qworacle as qo
from qwegn_amd import qwhip
from tests import helpers as H
from tests.test_gpu_attention import Case
from tests.test_gpu_heads import same

pytestmark = pytest.mark.gpu
HIDDEN, HEADS, KV, D, PAGE, PAGES, SEQS, MOST = 512, 8, 2, 64, 16, 24, 2, 96
WIDTH = (HEADS + 2 * KV) * D


@pytest.fixture(scope="module")
def dev():
    return qwhip.Device(0)


class Layer:
    def __init__(self, dev):
        self.dev, rng = dev, np.random.default_rng(7)
        blocks, self.w_qkv = H.make_bank("hq8_g32", WIDTH, HIDDEN, seed=1)
        self.qkv_bank = dev.put(blocks)
        self.qkv = H.view_of(dev, self.qkv_bank, "hq8_g32", WIDTH, HIDDEN)
        blocks, self.w_o = H.make_bank("hq4_g64", HIDDEN, HEADS * D, seed=2)
        self.o_bank = dev.put(blocks)
        self.o = H.view_of(dev, self.o_bank, "hq4_g64", HIDDEN, HEADS * D)
        self.gamma = (0.1 * rng.standard_normal(HIDDEN)).astype(np.float16)
        self.qk_gamma = (0.1 * rng.standard_normal((2, D))).astype(np.float16)
        self.table = qwkv.table(MOST, D)
        self.keep = [dev.put(a) for a in (self.gamma, self.qk_gamma[0], self.qk_gamma[1], self.table)]
        self.cache = qwkv.Cache(PAGES, PAGE, KV, D, fill=0xFF)
        self.pages = dev.put(self.cache.bytes)
        self.view = qwhip.KvCache(self.pages.ptr, self.cache.bytes.nbytes, PAGES, PAGE, KV, D)
        self.blocks = rng.permutation(PAGES)[: SEQS * MOST // PAGE].astype(np.int32).reshape(SEQS, -1)
        self.blocks_dev = dev.put(self.blocks)

    def rules(self, position):
        return qwhip.HeadRules(position=position, cos_sin=self.keep[3].ptr, q_gamma=self.keep[1].ptr, k_gamma=self.keep[2].ptr, positions=MOST, rope_dims=D, eps=1e-6,
                               flags=qwhip.HEAD_GAMMA_PLUS_ONE | qwhip.HEAD_FWHT_QK | qwhip.HEAD_FWHT_V)

    def slots(self, seq, token):
        return (self.blocks[seq, np.asarray(token) // PAGE] * PAGE + np.asarray(token) % PAGE).astype(np.int32)

    def check_step(self, qkv16, position, slots, q16, starts, lengths, out16, lse):
        """The steps behind the projection, each against its definition on what the one before it left."""
        rows = len(qkv16)
        x = qkv16.astype(np.float32).reshape(rows, -1, D)
        args = (True, 1e-6, self.table, position)
        q = qwkv.heads(x[:, :HEADS], self.qk_gamma[0], *args, fwht=True)
        k = qwkv.heads(x[:, HEADS:HEADS + KV], self.qk_gamma[1], *args, fwht=True)
        assert same(q16.reshape(q.shape), q.astype(np.float16), "f16")
        self.cache.put(slots, k, qwkv.fwht32(x[:, HEADS + KV:]))
        assert np.array_equal(self.pages.download(np.uint8, self.cache.bytes.shape), self.cache.bytes)
        case = Case.__new__(Case)
        case.d, case.heads, case.shared, case.t, case.window = D, KV, HEADS // KV, "f16", 0
        case.cache, case.table, case.q, case.scale = self.cache, self.blocks, q16.reshape(rows, HEADS, D), np.float32(D ** -0.5)
        case.start, case.lengths, case.seqs, case.total = np.asarray(starts), np.asarray(lengths), SEQS, rows
        case.check(out16.reshape(rows, HEADS, D), lse)


@pytest.fixture(scope="module")
def layer(dev):
    return Layer(dev)


def test_prompt_then_captured_decode(dev, layer):
    lib, main, rng = dev.lib, dev.stream, np.random.default_rng(8)
    first = [45, 20]
    rows = sum(first)
    starts = np.array([0, first[0], rows], np.int32)
    lengths = np.array(first, np.int32)
    position = np.concatenate([np.arange(n) for n in first]).astype(np.int32)
    slots = np.concatenate([layer.slots(s, np.arange(n)) for s, n in enumerate(first)])
    x = rng.standard_normal((rows, HIDDEN)).astype(np.float16)
    xb, pb, sb, stb, lb = (dev.put(a) for a in (x, position, slots, starts, lengths))
    normed, qkv, q, out, y = (dev.alloc(rows * n * 2) for n in (HIDDEN, WIDTH, HEADS * D, HEADS * D, HIDDEN))
    lse, room = dev.alloc(rows * HEADS * 4), dev.alloc(1 << 22)
    rules, tight, kv_at = layer.rules(pb.ptr), WIDTH, HEADS * D * 2
    batch = qwhip.KvBatch(stb.ptr, lb.ptr, layer.blocks_dev.ptr, layer.blocks.shape[1], SEQS, max(first), max(first))
    st = main.handle
    qwhip.check(lib.qwhip_rmsnorm(st, xb.ptr, layer.keep[0].ptr, None, rows, HIDDEN, 1e-6, 1, normed.ptr))
    qwhip.check(lib.qwhip_gemm(st, C.byref(layer.qkv), normed.ptr, qwhip.F16, rows, 0, qkv.ptr, qwhip.F16, 0, qwhip.X_PREROTATED, None, 0))
    qwhip.check(lib.qwhip_kv_append_mxfp4(st, C.byref(layer.view), C.byref(rules), rows, sb.ptr, qkv.ptr + kv_at, tight, qkv.ptr + kv_at + KV * D * 2, tight, qwhip.F16, qkv.ptr, HEADS, tight,
                                          q.ptr, 0, qwhip.F16, None, None))
    qwhip.check(lib.qwhip_kv_attention_mxfp4(st, C.byref(layer.view), C.byref(batch), q.ptr, qwhip.F16, HEADS, 0, rows, D ** -0.5, 0, out.ptr, 0, lse.ptr, room.ptr, room.nbytes))
    qwhip.check(lib.qwhip_gemm(st, C.byref(layer.o), out.ptr, qwhip.F16, rows, 0, y.ptr, qwhip.F16, 0, qwhip.X_PREROTATED, None, 0))
    main.sync()
    n16, p16 = normed.download(np.float16, (rows, HIDDEN)), qkv.download(np.float16, (rows, WIDTH))
    assert qo.normalized_error(p16, qo.matmul_ref_f64(n16, layer.w_qkv)) <= 2e-3
    o16 = out.download(np.float16, (rows, HEADS * D))
    layer.check_step(p16, position, slots, q.download(np.float16, (rows, HEADS * D)), starts, lengths, o16, lse.download(np.float32, (rows, HEADS)))
    assert qo.normalized_error(y.download(np.float16, (rows, HIDDEN)), qo.matmul_ref_f64(o16, layer.w_o)) <= 2e-3

    # decode: positions, slots and lengths live on the device; the graph is captured once
    stream = qwhip.Stream(dev)
    bufs = {n: dev.alloc(SEQS * w * 2) for n, w in (("x", HIDDEN), ("normed", HIDDEN), ("qkv", WIDTH), ("q", HEADS * D), ("out", HEADS * D), ("y", HIDDEN))}
    pos_d, slot_d, len_d = (dev.put(np.zeros(SEQS, np.int32)) for _ in range(3))
    step_rules = layer.rules(pos_d.ptr)
    grown = qwhip.KvBatch(None, len_d.ptr, layer.blocks_dev.ptr, layer.blocks.shape[1], SEQS, 1, MOST)
    s = stream.handle

    def step():
        b = {n: v.ptr for n, v in bufs.items()}
        qwhip.check(lib.qwhip_rmsnorm(s, b["x"], layer.keep[0].ptr, None, SEQS, HIDDEN, 1e-6, 1, b["normed"]))
        qwhip.check(lib.qwhip_gemv(s, C.byref(layer.qkv), b["normed"], qwhip.F16, SEQS, qwhip.X_PREROTATED, b["qkv"], None))
        qwhip.check(lib.qwhip_kv_append_mxfp4(s, C.byref(layer.view), C.byref(step_rules), SEQS, slot_d.ptr, b["qkv"] + kv_at, tight, b["qkv"] + kv_at + KV * D * 2, tight, qwhip.F16,
                                              b["qkv"], HEADS, tight, b["q"], 0, qwhip.F16, None, None))
        qwhip.check(lib.qwhip_kv_attention_mxfp4(s, C.byref(layer.view), C.byref(grown), b["q"], qwhip.F16, HEADS, 0, SEQS, D ** -0.5, 0, b["out"], 0, lse.ptr, room.ptr, room.nbytes))
        qwhip.check(lib.qwhip_gemv(s, C.byref(layer.o), b["out"], qwhip.F16, SEQS, qwhip.X_PREROTATED, b["y"], None))

    graph = qwhip.Graph(stream, step)
    for turn in range(12):
        position = lengths.copy()
        slots = np.array([layer.slots(i, position[i]) for i in range(SEQS)], np.int32)
        if turn == 7:
            slots[1] = -1                                                                 # a request that has left: its row is padding
        lengths = lengths + (slots >= 0)
        for b, a in ((pos_d, position), (slot_d, slots), (len_d, lengths), (bufs["x"], rng.standard_normal((SEQS, HIDDEN)).astype(np.float16))):
            b.upload(a.astype(np.int32) if a.dtype != np.float16 else a)
        q_before = bufs["q"].download(np.float16, (SEQS, HEADS * D))
        graph.launch()
        stream.sync()
        got = {n: b.download(np.float16, (SEQS, b.nbytes // (2 * SEQS))) for n, b in bufs.items()}
        assert qo.normalized_error(got["qkv"], qo.matmul_ref_f64(got["normed"], layer.w_qkv)) <= 2e-3
        assert qo.normalized_error(got["y"], qo.matmul_ref_f64(got["out"], layer.w_o)) <= 2e-3
        if turn == 7:
            assert np.array_equal(got["q"][1], q_before[1])                               # nothing written for it
            x = got["qkv"][:1].astype(np.float32).reshape(1, -1, D)
            args = (True, 1e-6, layer.table, position[:1])
            layer.cache.put(slots[:1], qwkv.heads(x[:, HEADS:HEADS + KV], layer.qk_gamma[1], *args, fwht=True), qwkv.fwht32(x[:, HEADS + KV:]))
            assert np.array_equal(layer.pages.download(np.uint8, layer.cache.bytes.shape), layer.cache.bytes)
            continue
        layer.check_step(got["qkv"], position, slots, got["q"], np.arange(SEQS + 1), lengths, got["out"], lse.download(np.float32, (rows, HEADS))[:SEQS])
    graph.destroy()
    for b in (xb, pb, sb, stb, lb, normed, qkv, q, out, y, lse, room, pos_d, slot_d, len_d, *bufs.values()):
        b.free()


def test_transformed_values_come_out_in_the_banks_basis(dev):
    """The same values with and without the transform, under equal weights (keys of zero): one output is the transform of the other, up to what four bits leave.
    An element is off by at most a quarter of its block's largest (8 - 6 of 8 units), so a block's mean by sqrt(32) / 4 of the largest there is, in either
    basis (the transform keeps lengths); f16 weights and outputs add 2^-10 of that largest."""
    rng = np.random.default_rng(9)
    n, d = 200, 128
    v = rng.standard_normal((n, 1, d))
    outs, bound = [], 0.0
    for turned in (False, True):
        c = Case(dev, 1, d, 1, 4, 16, [1], [n], "f16", noise=False)
        t = np.arange(n)
        u = (qwkv.fwht32(v) if turned else v).astype(np.float32)
        c.cache.put(c.table[0][t // 16] * 16 + t % 16, np.zeros_like(u), u)
        y, l = c.run()
        c.check(y, l)
        outs.append(y[0].astype(np.float64))
        bound += np.sqrt(32.0) * (0.25 + 2.0 ** -10) * np.abs(u).max()
    off = (qwkv.fwht32(outs[1]) - outs[0]).reshape(-1, 32)
    assert (np.linalg.norm(off, axis=1) <= bound).all()
    assert np.linalg.norm(outs[1] - outs[0]) > 0.5 * np.linalg.norm(outs[0])               # and the bases do differ
