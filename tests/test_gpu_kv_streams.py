"""The doors between the q|k|v projection and the output projection with calls in flight on two streams: everything is enqueued on both before either is waited for, and each call has buffers and
a workspace of its own."""
import ctypes as C

import numpy as np
import pytest

from oracle import qwkv
from qwegn_amd import qwhip
from tests.test_gpu_attention import Case
from tests.test_gpu_heads import Rules, encode

pytestmark = pytest.mark.gpu
CALLS = 6


@pytest.fixture(scope="module")
def dev():
    return qwhip.Device(0)


def together(dev, jobs):
    """jobs: (call(stream), outputs).  One after the other on one stream, then in turn on two streams with the outputs cleared: the same bits."""
    streams = [dev.stream, qwhip.Stream(dev)]

    def clear():
        for _, outs in jobs:
            for b in outs:
                qwhip.check(dev.lib.qwhip_fill_u32(dev.stream.handle, b.ptr, 0x7E017E01, b.nbytes // 4))
        dev.stream.sync()

    def take():
        return [[b.download(np.uint32, (b.nbytes // 4,)) for b in outs] for _, outs in jobs]

    clear()
    for call, _ in jobs:
        call(dev.stream)
        dev.stream.sync()
    want = take()
    for turn in range(3):
        clear()
        for i, (call, _) in enumerate(jobs):
            call(streams[(i + turn) % 2])
        for s in streams:
            s.sync()
        for i, (a, b) in enumerate(zip(take(), want)):
            assert all(np.array_equal(x, y) for x, y in zip(a, b)), (turn, i)
    return want


@pytest.mark.parametrize("rows,length,shared,d,bound", [([1], 6000, 4, 128, 6000), ([1] * 5, 3000, 4, 64, 3000), ([9], 5000, 4, 256, 5000), ([70], 2000, 4, 128, 1 << 20)])
def test_attention(dev, rows, length, shared, d, bound):
    keep, jobs, cases = [], [], []
    for i in range(CALLS):
        c = Case(dev, 100 + i, d, 2, shared, 64, rows, [length - 7 * s for s in range(len(rows))], "bf16")
        heads, table = 2 * shared, np.zeros((len(rows), -(-bound // 64)), np.int32)
        table[:, : c.each] = c.table
        bufs = [dev.put(a) for a in (c.q, c.cache.bytes, c.start, c.lengths.astype(np.int32), table)]
        view = qwhip.KvCache(bufs[1].ptr, c.cache.bytes.nbytes, len(c.cache.bytes), 64, 2, d)
        batch = qwhip.KvBatch(bufs[2].ptr, bufs[3].ptr, bufs[4].ptr, table.shape[1], len(rows), max(rows), bound)
        need = dev.lib.qwhip_kv_attention_workspace_bytes(C.byref(view), C.byref(batch), heads, c.total, 0)
        assert need > 0                                                                   # in parts: the workspace is used
        out, lse, ws = dev.alloc(c.q.nbytes), dev.alloc(c.total * heads * 4), dev.alloc(need)

        def call(st, c=c, b=bufs, view=view, batch=batch, out=out, lse=lse, ws=ws, heads=heads):
            qwhip.check(dev.lib.qwhip_kv_attention_mxfp4(st.handle, C.byref(view), C.byref(batch), b[0].ptr, qwhip.BF16, heads, 0, c.total, c.scale, 0, out.ptr, 0, lse.ptr, ws.ptr, ws.nbytes))

        jobs.append((call, [out, lse]))
        cases.append(c)
        keep += [*bufs, out, lse, ws]
    for c, (out, lse) in zip(cases, together(dev, jobs)):
        c.check(out.view(np.uint16).reshape(c.q.shape), lse.view(np.float32).reshape(c.total, -1))
    for b in keep:
        b.free()


@pytest.mark.parametrize("rows", [3, 300, 2500])
def test_heads_and_cache(dev, rows):
    d, qh, kh, page, keep, jobs = 128, 8, 2, 32, [], []
    ld = (qh + 2 * kh) * d
    for i in range(CALLS):
        rng = np.random.default_rng(200 + i)
        rules = Rules(dev, rng, d, rows, 128, qwkv.PLUS_ONE | qwkv.FWHT_QK | (qwkv.FWHT_V if i % 2 else 0))
        pages = rows // page + 1
        size = pages * dev.lib.qwhip_kv_page_bytes(page, kh, d)
        x, slots = dev.put(encode(rng.standard_normal((rows, ld)), "bf16")), dev.put(rng.permutation(pages * page)[:rows].astype(np.int32))
        outs = [dev.alloc(n) for n in (size, rows * qh * d * 2, rows * kh * d * 2, rows * kh * d * 2)]
        view, k = qwhip.KvCache(outs[0].ptr, size, pages, page, kh, d), x.ptr + qh * d * 2

        def call(st, i=i, x=x, slots=slots, outs=outs, view=view, k=k, rules=rules):
            if i % 2:
                qwhip.check(dev.lib.qwhip_kv_append_mxfp4(st.handle, C.byref(view), C.byref(rules.c), rows, slots.ptr, k, ld, k + kh * d * 2, ld, qwhip.BF16, x.ptr, qh, ld, outs[1].ptr, 0,
                                                          qwhip.BF16, outs[2].ptr, outs[3].ptr))
            else:
                qwhip.check(dev.lib.qwhip_head_norm_rope(st.handle, C.byref(rules.c), rows, d, x.ptr, qh, ld, k, kh, ld, qwhip.BF16, outs[1].ptr, 0, outs[2].ptr, 0, qwhip.BF16))

        jobs.append((call, outs))
        keep += [x, slots, *outs]
    together(dev, jobs)
    for b in keep:
        b.free()
