"""What the doors between the q|k|v projection and the output projection refuse, on a host without a GPU: every check runs before the stream is looked at,
so a block of zeros stands for the stream and host addresses for device memory."""
import ctypes as C

import pytest

from qwegn_amd import qwhip

_store = (C.c_uint8 * (1 << 16))()
BASE = (C.addressof(_store) + 255) // 256 * 256
STREAM = (C.c_uint8 * 4096)()
ST = C.addressof(STREAM)


@pytest.fixture(scope="module")
def lib():
    return qwhip.load()


def cache(**kw):
    a = dict(pages=BASE, bytes=1 << 30, page_count=8, page_size=16, kv_heads=2, head_dim=64)
    a.update(kw)
    return qwhip.KvCache(**a)


def test_page_bytes_and_view(lib):
    for page in (16, 32, 64, 128, 256):
        for d in (64, 128, 256):
            assert lib.qwhip_kv_page_bytes(page, 3, d) == page * 3 * (d // 2 + d // 32) * 2
    for bad in ((0, 1, 64), (8, 1, 64), (48, 1, 64), (512, 1, 64), (16, 0, 64), (16, 1025, 64), (16, 1, 32), (16, 1, 96), (16, 1, 512), (16, 1, 0)):
        assert lib.qwhip_kv_page_bytes(*bad) == 0, bad
    ok = lambda **kw: lib.qwhip_kv_cache_validate(C.byref(cache(**kw)))  # noqa: E731
    need = 8 * lib.qwhip_kv_page_bytes(16, 2, 64)
    assert ok() == ok(bytes=need) == qwhip.OK
    assert ok(bytes=need - 1) == qwhip.E_BAD_WEIGHTS and b"bytes" in lib.qwhip_last_error()
    assert ok(page_count=(1 << 27) - 1, bytes=1 << 60) == qwhip.OK
    for bad in (dict(page_count=0), dict(page_count=1 << 27, bytes=1 << 60), dict(page_size=24), dict(kv_heads=0), dict(head_dim=96), dict(pages=BASE + 8)):
        assert ok(**bad) == qwhip.E_BAD_WEIGHTS, bad
    assert ok(pages=None) == qwhip.E_NULL and lib.qwhip_kv_cache_validate(None) == qwhip.E_NULL


def rules(**kw):
    a = dict(position=BASE, cos_sin=BASE, q_gamma=BASE, k_gamma=BASE, positions=4, rope_dims=32, eps=1e-6, flags=0)
    a.update(kw)
    return qwhip.HeadRules(**a)


BAD_RULES = [(dict(position=None), qwhip.E_NULL), (dict(positions=0), qwhip.E_BAD_SHAPE), (dict(positions=1 << 31), qwhip.E_BAD_SHAPE), (dict(rope_dims=0), qwhip.E_BAD_SHAPE),
             (dict(rope_dims=24), qwhip.E_BAD_SHAPE), (dict(rope_dims=80), qwhip.E_BAD_SHAPE), (dict(flags=16), qwhip.E_BAD_SHAPE), (dict(eps=-1.0), qwhip.E_BAD_SHAPE),
             (dict(eps=float("nan")), qwhip.E_BAD_SHAPE), (dict(eps=float("inf")), qwhip.E_BAD_SHAPE), (dict(cos_sin=BASE + 4), qwhip.E_BAD_SHAPE),
             (dict(q_gamma=BASE + 2), qwhip.E_BAD_SHAPE), (dict(k_gamma=BASE + 2), qwhip.E_BAD_SHAPE)]


def norm_rope(lib, r=None, **kw):
    a = dict(s=ST, rows=3, d=64, q=BASE, qh=2, ldq=0, k=BASE, kh=1, ldk=0, t=qwhip.F16, qo=BASE + 4096, ldqo=0, ko=BASE + 8192, ldko=0, o=qwhip.F16)
    a.update(kw)
    r = rules() if r is None else r
    return lib.qwhip_head_norm_rope(a["s"], C.byref(r) if r else None, a["rows"], a["d"], a["q"], a["qh"], a["ldq"], a["k"], a["kh"], a["ldk"], a["t"], a["qo"], a["ldqo"], a["ko"],
                                    a["ldko"], a["o"])


@pytest.mark.parametrize("change,want", BAD_RULES + [(dict(flags=qwhip.HEAD_FWHT_V), qwhip.E_BAD_SHAPE)])
def test_rules_of_norm_rope(lib, change, want):
    assert norm_rope(lib, rules(**change)) == want, change


@pytest.mark.parametrize("change,want", [
    (dict(s=None), qwhip.E_NULL), (dict(r=False), qwhip.E_NULL), (dict(q=None), qwhip.E_NULL), (dict(k=None), qwhip.E_NULL), (dict(qo=None), qwhip.E_NULL),
    (dict(ko=None), qwhip.E_NULL), (dict(t=qwhip.I32), qwhip.E_BAD_SHAPE), (dict(o=9), qwhip.E_BAD_SHAPE), (dict(d=0), qwhip.E_BAD_SHAPE), (dict(d=48), qwhip.E_BAD_SHAPE),
    (dict(d=288), qwhip.E_BAD_SHAPE), (dict(rows=1 << 24), qwhip.E_BAD_SHAPE), (dict(qh=65536), qwhip.E_BAD_SHAPE), (dict(ldq=120), qwhip.E_BAD_SHAPE),
    (dict(ldq=132), qwhip.E_BAD_SHAPE), (dict(t=qwhip.F32, ldq=130), qwhip.E_BAD_SHAPE), (dict(ldqo=64), qwhip.E_BAD_SHAPE), (dict(ldko=68), qwhip.E_BAD_SHAPE),
    (dict(q=BASE + 8), qwhip.E_BAD_SHAPE), (dict(ko=BASE + 2), qwhip.E_BAD_SHAPE), (dict(qo=BASE, o=qwhip.BF16), qwhip.E_BAD_SHAPE), (dict(qo=BASE, ldqo=136), qwhip.E_BAD_SHAPE),
    (dict(ko=BASE, t=qwhip.F32), qwhip.E_BAD_SHAPE),
])
def test_norm_rope(lib, change, want):
    assert norm_rope(lib, **change) == want, change


def test_nothing_to_do(lib):
    assert norm_rope(lib, rows=0, q=None, k=None, qo=None, ko=None) == qwhip.OK
    assert norm_rope(lib, qh=0, kh=0, q=None, k=None, qo=None, ko=None) == qwhip.OK
    assert append(lib, rows=0, slots=None, k=None, v=None) == qwhip.OK
    assert attention(lib, rows=0, batch=batch(seqs=2)) == qwhip.OK
    assert attention(lib, batch=batch(seqs=0)) == qwhip.OK
    assert attention(lib, batch=batch(max_rows=0)) == qwhip.OK


def append(lib, c=None, r=None, **kw):
    a = dict(s=ST, rows=3, slots=BASE, k=BASE, ldk=0, v=BASE, ldv=0, t=qwhip.BF16, q=BASE, qh=4, ldq=0, qo=BASE + 4096, ldqo=0, o=qwhip.BF16, kv=None, vv=None)
    a.update(kw)
    c = cache() if c is None else c
    return lib.qwhip_kv_append_mxfp4(a["s"], C.byref(c) if c else None, C.byref(r) if r else None, a["rows"], a["slots"], a["k"], a["ldk"], a["v"], a["ldv"], a["t"], a["q"], a["qh"],
                                     a["ldq"], a["qo"], a["ldqo"], a["o"], a["kv"], a["vv"])


@pytest.mark.parametrize("change,want", BAD_RULES)
def test_rules_of_append(lib, change, want):
    assert append(lib, r=rules(**change)) == want, change


@pytest.mark.parametrize("change,want", [
    (dict(s=None), qwhip.E_NULL), (dict(c=False), qwhip.E_NULL), (dict(slots=None), qwhip.E_NULL), (dict(k=None), qwhip.E_NULL), (dict(v=None), qwhip.E_NULL),
    (dict(q=None), qwhip.E_NULL), (dict(qo=None), qwhip.E_NULL), (dict(t=3), qwhip.E_BAD_SHAPE), (dict(o=3), qwhip.E_BAD_SHAPE), (dict(qh=0, o=3, kv=BASE), qwhip.E_BAD_SHAPE),
    (dict(rows=1 << 24), qwhip.E_BAD_SHAPE), (dict(ldk=64), qwhip.E_BAD_SHAPE), (dict(ldv=130), qwhip.E_BAD_SHAPE), (dict(ldq=264, qo=BASE), qwhip.E_BAD_SHAPE),
    (dict(k=BASE + 8), qwhip.E_BAD_SHAPE), (dict(kv=BASE + 8), qwhip.E_BAD_SHAPE), (dict(vv=BASE + 2), qwhip.E_BAD_SHAPE), (dict(c=cache(bytes=10)), qwhip.E_BAD_WEIGHTS),
    (dict(c=cache(head_dim=32)), qwhip.E_BAD_WEIGHTS),
])
def test_append(lib, change, want):
    assert append(lib, **change) == want, change


def batch(**kw):
    a = dict(row_start=BASE, lengths=BASE, block_table=BASE, ld_table=4, seqs=2, max_rows=3, max_length=64)
    a.update(kw)
    return qwhip.KvBatch(**a)


def attention(lib, c=None, **kw):
    a = dict(s=ST, q=BASE, t=qwhip.F16, qh=4, ldq=0, rows=5, scale=0.125, window=0, out=BASE + 8192, ldo=0, lse=None, ws=None, wsb=0)
    a.update(kw)
    c = cache() if c is None else c
    b = a.pop("batch", batch())
    return lib.qwhip_kv_attention_mxfp4(a["s"], C.byref(c) if c else None, C.byref(b) if b else None, a["q"], a["t"], a["qh"], a["ldq"], a["rows"], a["scale"], a["window"], a["out"],
                                        a["ldo"], a["lse"], a["ws"], a["wsb"])


@pytest.mark.parametrize("change,want", [
    (dict(s=None), qwhip.E_NULL), (dict(c=False), qwhip.E_NULL), (dict(batch=None), qwhip.E_NULL), (dict(q=None), qwhip.E_NULL), (dict(out=None), qwhip.E_NULL),
    (dict(batch=batch(lengths=None)), qwhip.E_NULL), (dict(batch=batch(block_table=None)), qwhip.E_NULL), (dict(t=qwhip.F32), qwhip.E_BAD_SHAPE), (dict(qh=0), qwhip.E_BAD_SHAPE),
    (dict(qh=3), qwhip.E_BAD_SHAPE), (dict(qh=65536), qwhip.E_BAD_SHAPE), (dict(scale=0.0), qwhip.E_BAD_SHAPE), (dict(scale=-1.0), qwhip.E_BAD_SHAPE),
    (dict(scale=float("nan")), qwhip.E_BAD_SHAPE), (dict(scale=float("inf")), qwhip.E_BAD_SHAPE), (dict(ldq=128), qwhip.E_BAD_SHAPE), (dict(ldo=260), qwhip.E_BAD_SHAPE),
    (dict(q=BASE + 2), qwhip.E_BAD_SHAPE), (dict(out=BASE + 8), qwhip.E_BAD_SHAPE), (dict(ws=BASE + 4, wsb=100), qwhip.E_BAD_SHAPE), (dict(batch=batch(max_length=65)), qwhip.E_BAD_SHAPE),
    (dict(batch=batch(max_length=1 << 31, ld_table=1 << 30)), qwhip.E_BAD_SHAPE), (dict(batch=batch(seqs=65536)), qwhip.E_BAD_SHAPE), (dict(batch=batch(row_start=None)), qwhip.E_BAD_SHAPE),
    (dict(rows=1 << 31), qwhip.E_BAD_SHAPE), (dict(rows=1 << 30, batch=batch(max_rows=1 << 30)), qwhip.E_BAD_SHAPE), (dict(c=cache(page_size=8)), qwhip.E_BAD_WEIGHTS),
])
def test_attention(lib, change, want):
    assert attention(lib, **change) == want, change


@pytest.mark.parametrize("scale,want", [(2.0 ** -149, qwhip.OK), (2.0 ** 127 * 0.99, qwhip.OK), (2.0 ** 127 * 1.4, qwhip.E_BAD_SHAPE), (3.4e38, qwhip.E_BAD_SHAPE)])
def test_scales_of_scores(lib, scale, want):
    assert attention(lib, scale=scale, batch=batch(seqs=0)) == want


def test_workspace_bytes(lib):
    size = lambda c=cache(), b=batch(), qh=4, rows=5, window=0: lib.qwhip_kv_attention_workspace_bytes(C.byref(c), C.byref(b), qh, rows, window)  # noqa: E731
    long = batch(seqs=1, max_rows=1, max_length=1 << 17, ld_table=1 << 13)
    one = size(b=long, rows=1)
    assert one > 0 and one % (4 * (64 + 2) * 4) == 0
    assert size(b=long, rows=1, window=300) < one
    assert size(b=batch(max_length=0)) == 0 and size(rows=0) == 0 and size(qh=3) == 0
    assert size(b=batch(max_rows=1 << 20, max_length=64), rows=1 << 20) == 0        # rows enough for every compute unit
