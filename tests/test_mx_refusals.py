"""What the MXFP4 doors and qwhip_logits_process refuse, on a host without a GPU: every check runs before the stream is looked at, so a
block of zeros stands for the stream and host addresses for device memory."""
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


def view(n=8, k=64, ld=0, codes=BASE, scales=BASE + 8192, cb=4096, sb=4096):
    return qwhip.Mxfp4View(codes, scales, cb, sb, n, k, ld)


def test_view(lib):
    ok = lambda **kw: lib.qwhip_mxfp4_view_validate(C.byref(view(**kw)))  # noqa: E731
    assert ok() == qwhip.OK
    assert ok(cb=8 * 32, sb=8 * 2) == qwhip.OK
    assert ok(cb=8 * 32 - 1) == qwhip.E_BAD_WEIGHTS and b"planes" in lib.qwhip_last_error()
    assert ok(sb=8 * 2 - 1) == qwhip.E_BAD_WEIGHTS
    assert ok(ld=128, cb=7 * 64 + 32, sb=7 * 4 + 2) == qwhip.OK            # the last row ends with its columns
    assert ok(ld=128, cb=7 * 64 + 31) == qwhip.E_BAD_WEIGHTS
    for bad in (dict(n=0), dict(k=0), dict(k=48), dict(ld=32), dict(ld=80), dict(codes=BASE + 8), dict(n=0xFFFFFFFF, k=0xFFFFFFE0)):
        assert ok(**bad) == qwhip.E_BAD_WEIGHTS, bad
    assert ok(codes=None) == qwhip.E_NULL and ok(scales=None) == qwhip.E_NULL
    assert ok(scales=BASE + 8193) == qwhip.OK
    assert lib.qwhip_mxfp4_view_validate(None) == qwhip.E_NULL


@pytest.mark.parametrize("change,want", [
    (dict(s=None), qwhip.E_NULL), (dict(src=None), qwhip.E_NULL), (dict(codes=None), qwhip.E_NULL), (dict(scales=None), qwhip.E_NULL),
    (dict(k=0), qwhip.E_BAD_SHAPE), (dict(k=40), qwhip.E_BAD_SHAPE), (dict(ld=32), qwhip.E_BAD_SHAPE), (dict(ld=66), qwhip.E_BAD_SHAPE),
    (dict(t=qwhip.F32, ld=66), qwhip.E_BAD_SHAPE), (dict(ld=68), qwhip.E_BAD_SHAPE), (dict(t=qwhip.I32), qwhip.E_BAD_SHAPE), (dict(t=9), qwhip.E_BAD_SHAPE),
    (dict(src=BASE + 8), qwhip.E_BAD_SHAPE), (dict(codes=BASE + 4), qwhip.E_BAD_SHAPE), (dict(values=BASE + 2), qwhip.E_BAD_SHAPE),
    (dict(rows=0xFFFFFFFF, k=0xFFFFFFE0), qwhip.E_BAD_SHAPE), (dict(rows=1 << 20, k=1 << 15), qwhip.E_BAD_SHAPE), (dict(rows=0), qwhip.OK), (dict(rows=0, src=None), qwhip.OK)])
def test_quantise(lib, change, want):
    a = dict(s=ST, src=BASE, t=qwhip.F16, rows=4, k=64, ld=0, codes=BASE + 4096, scales=BASE + 8192, values=BASE + 16384) | change
    assert lib.qwhip_quantize_mxfp4(a["s"], a["src"], a["t"], a["rows"], a["k"], a["ld"], a["codes"], a["scales"], a["values"]) == want


def test_dequant(lib):
    v = view()
    assert lib.qwhip_dequant_mxfp4(None, C.byref(v), BASE, 0) == qwhip.E_NULL
    assert lib.qwhip_dequant_mxfp4(ST, None, BASE, 0) == qwhip.E_NULL
    assert lib.qwhip_dequant_mxfp4(ST, C.byref(v), None, 0) == qwhip.E_NULL
    assert lib.qwhip_dequant_mxfp4(ST, C.byref(v), BASE + 4, 0) == qwhip.E_BAD_SHAPE
    assert lib.qwhip_dequant_mxfp4(ST, C.byref(v), BASE, 3) == qwhip.E_BAD_SHAPE
    assert lib.qwhip_dequant_mxfp4(ST, C.byref(view(k=33)), BASE, 0) == qwhip.E_BAD_WEIGHTS
    assert lib.qwhip_dequant_mxfp4(ST, C.byref(view(n=1 << 20, k=1 << 15, cb=1 << 40, sb=1 << 40)), BASE, 0) == qwhip.E_BAD_SHAPE


@pytest.mark.parametrize("change,want", [
    (dict(s=None), qwhip.E_NULL), (dict(w=None), qwhip.E_NULL), (dict(x=None), qwhip.E_NULL), (dict(y=None), qwhip.E_NULL),
    (dict(w=view(k=48)), qwhip.E_BAD_WEIGHTS), (dict(x=view(k=96)), qwhip.E_BAD_SHAPE), (dict(t=3), qwhip.E_BAD_SHAPE), (dict(ldy=7), qwhip.E_BAD_SHAPE),
    (dict(y=BASE + 2), qwhip.E_BAD_SHAPE), (dict(t=qwhip.BF16, y=BASE + 1), qwhip.E_BAD_SHAPE), (dict(ws=BASE + 8, wb=4096), qwhip.E_BAD_SHAPE),
    (dict(x=view(n=0)), qwhip.OK), (dict(x=view(n=0, k=32)), qwhip.E_BAD_SHAPE)])
def test_gemm(lib, change, want):
    a = dict(s=ST, w=view(), x=view(n=3), y=BASE + 16384, t=qwhip.F32, ldy=0, ws=None, wb=0) | change
    ref = lambda v: C.byref(v) if v is not None else None  # noqa: E731
    assert lib.qwhip_mxfp4_gemm(a["s"], ref(a["w"]), ref(a["x"]), a["y"], a["t"], a["ldy"], a["ws"], a["wb"]) == want


@pytest.mark.parametrize("change,want", [
    (dict(s=None), qwhip.E_NULL), (dict(w=None), qwhip.E_NULL), (dict(x=None), qwhip.E_NULL), (dict(y16=None, y32=None), qwhip.E_NULL),
    (dict(w=view(k=48)), qwhip.E_BAD_WEIGHTS), (dict(t=qwhip.F32), qwhip.E_BAD_SHAPE), (dict(m=17), qwhip.E_BAD_SHAPE), (dict(x=BASE + 8), qwhip.E_BAD_SHAPE),
    (dict(y16=BASE + 1), qwhip.E_BAD_SHAPE), (dict(y32=BASE + 2), qwhip.E_BAD_SHAPE), (dict(m=0), qwhip.OK)])
def test_gemv(lib, change, want):
    a = dict(s=ST, w=view(), x=BASE, t=qwhip.F16, m=2, y16=BASE + 16384, y32=BASE + 20480) | change
    assert lib.qwhip_mxfp4_gemv(a["s"], C.byref(a["w"]) if a["w"] is not None else None, a["x"], a["t"], a["m"], a["y16"], a["y32"]) == want


@pytest.mark.parametrize("change,rules,want", [
    (dict(s=None), {}, qwhip.E_NULL), (dict(logits=None), {}, qwhip.E_NULL), (dict(out=None, tokens=None), {}, qwhip.E_NULL),
    (dict(t=3), {}, qwhip.E_BAD_SHAPE), (dict(n=0), {}, qwhip.E_BAD_SHAPE), (dict(n=1 << 30), {}, qwhip.E_BAD_SHAPE), (dict(ld=99), {}, qwhip.E_BAD_SHAPE),
    (dict(ld_out=99), {}, qwhip.E_BAD_SHAPE), (dict(rows=65536), {}, qwhip.E_BAD_SHAPE), (dict(logits=BASE + 2), {}, qwhip.E_BAD_SHAPE),
    (dict(out=BASE + 4097), {}, qwhip.E_BAD_SHAPE), (dict(out=BASE, ld_out=104), {}, qwhip.E_BAD_SHAPE), (dict(ws=None), {}, qwhip.E_NULL),
    (dict(wb=15), {}, qwhip.E_BAD_SHAPE), (dict(ws=BASE + 8196), {}, qwhip.E_BAD_SHAPE), (dict(rows=0), {}, qwhip.OK),
    ({}, dict(history=BASE, ld_history=4), qwhip.E_NULL), ({}, dict(history=BASE, total_len=BASE, ld_history=1 << 30), qwhip.E_BAD_SHAPE),
    ({}, dict(bias_off=BASE, bias_count=2, bias_tok=BASE), qwhip.E_NULL), ({}, dict(bias_off=BASE, bias_count=2, bias_val=BASE), qwhip.E_NULL),
    ({}, dict(allowed=BASE, allowed_rows=1, ld_allowed=3), qwhip.E_BAD_SHAPE)])
def test_logits(lib, change, rules, want):
    a = dict(s=ST, logits=BASE, t=qwhip.F32, rows=2, n=100, ld=0, out=BASE + 4096, ld_out=0, tokens=BASE + 12288, ws=BASE + 8192, wb=4096) | change
    r = qwhip.LogitsRules(**rules)
    assert lib.qwhip_logits_process(a["s"], C.byref(r), a["logits"], a["t"], a["rows"], a["n"], a["ld"], a["out"], a["ld_out"], a["tokens"], a["ws"], a["wb"]) == want
    assert lib.qwhip_logits_process(ST, None, BASE, 0, 2, 100, 0, BASE, 0, None, None, 0) == qwhip.E_NULL
