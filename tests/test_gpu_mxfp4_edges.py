"""MXFP4 products where they can go wrong: scales at the ends of their range, operands of very many rows, every kernel form in its steady loop,
and data whose sums fp32 holds exactly, so that one element out of a long row shows."""
import ctypes as C

import numpy as np
import pytest

from oracle import qwmx
from oracle import qworacle as qo
from qwegn_amd import qwhip
from tests.test_gpu_mxfp4 import as_type, check_product, filled, free, gemm, gemv, put_bank, random_bank

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return qwhip.Device(0)


@pytest.mark.parametrize("t", [qwhip.F16, qwhip.BF16])
@pytest.mark.parametrize("m,n,k", [(1, 33, 672), (6, 50, 1024), (9, 40, 17408)])
@pytest.mark.parametrize("where", ["253", "254", "both among others", "one block"])
def test_gemv_scales_that_reach_past_bf16(dev, t, m, n, k, where):
    """Elements of 2^128 and on, which neither bf16 nor fp32 holds: their products with small activations are finite, those with a zero are zero."""
    bank = random_bank(n, k, 31)
    scales = bank[1]
    if where in ("253", "254"):
        scales[:] = int(where)
    elif where == "one block":
        scales[n // 2, (k // 32) // 2] = 254
    else:
        scales[::3, ::2], scales[1::3, 1::5] = 254, 253
    image, val = as_type(np.random.default_rng(m).standard_normal((m, k)) * 2.0 ** -14, t)
    image[:, ::7], val[:, ::7] = 0, 0
    if m > 1:
        image[m // 2], val[m // 2] = 0, 0
    w = qwmx.values(bank[0], scales)
    wv, bufs = put_bank(dev, (bank[0], scales, None), k)
    _, y32 = gemv(dev, wv, image, t, m, n)
    assert m == 1 or np.array_equal(y32[m // 2], np.zeros(n, np.float32))
    check_product(y32, val.astype(np.float64), w, qwhip.F32)
    free(*bufs)


def test_gemv_nan_block_beside_scales_that_reach_past_bf16(dev):
    n, k, m = 40, 1056, 3
    bank = random_bank(n, k, 37)
    bank[1][:, 4] = 254
    bank[1][11, 4] = bank[1][12, 32] = 255
    image, val = as_type(np.random.default_rng(2).standard_normal((m, k)) * 2.0 ** -20, qwhip.BF16)
    w = qwmx.values(bank[0], bank[1])
    wv, bufs = put_bank(dev, (bank[0], bank[1], None), k)
    _, y32 = gemv(dev, wv, image, qwhip.BF16, m, n)
    nan = np.zeros((m, n), bool)
    nan[:, 11:13] = True
    assert np.array_equal(np.isnan(y32), nan)
    w[11:13] = 0.0
    check_product(np.where(nan, 0.0, y32), val.astype(np.float64), w, qwhip.F32)
    free(*bufs)


@pytest.mark.parametrize("n,ldy,t", [(5, 7, qwhip.F32), (33, 0, qwhip.BF16), (130, 0, qwhip.BF16)])
def test_gemm_of_millions_of_rows(dev, n, ldy, t):
    """More rows than the second dimension of a grid has tiles of: every row is there, checked at both ends and about the seam."""
    m, k = 65535 * 32 + 70, 32
    wb, xb = random_bank(n, k, 1), random_bank(m, k, 2, ld=64)
    wv, b0 = put_bank(dev, wb, k)
    xv, b1 = put_bank(dev, xb, k)
    got = gemm(dev, wv, xv, m, n, t, ldy=ldy)
    for at in (0, m // 2, m - 600, m - 300):
        check_product(got[at:at + 300], xb[2][at:at + 300], wb[2], t)
    free(*b0, *b1)


# ---- data whose sums are exact ---------------------------------------------------------------------------------------------------------
# Elements are multiples of a unit u, and so are products and all partial sums; where sum |x w| stays under 2^24 u every one of them is an fp32
# number, in whatever order they are added: the results have to be equal.  One block, piece or scale out of place changes almost every one.
def exact_bank(n, k, seed, scale_bytes, ld=None):
    """Every code under scales drawn from `scale_bytes`; (codes, scales, values f32): multiples of half the smallest scale."""
    rng = np.random.default_rng(seed)
    ld = ld or k
    codes = rng.integers(0, 256, (n, ld // 2), dtype=np.uint8)
    scales = rng.choice(np.array(scale_bytes, np.uint8), (n, ld // 32))
    with np.errstate(over="ignore"):
        return codes, scales, qwmx.values(codes[:, :k // 2], scales[:, :k // 32]).astype(np.float32)


def exact_product(x, w, unit):
    assert (np.abs(x) @ np.abs(w).T).max() < 2.0 ** 24 * unit
    return x @ w.T


GEMV_EXACT = [(1, 20, 90112), (1, 37, 90240), (2, 35, 33312), (2, 500, 33280), (3, 70, 22048), (5, 333, 17408), (8, 96, 7712), (9, 333, 17440), (16, 4200, 8224), (13, 64, 4640), (9, 4096, 8768), (16, 4095, 8704), (12, 4097, 8736),   # chunks
              (1, 40007, 64), (4, 17001, 544), (7, 9000, 2592), (3, 5000, 3616), (1, 640, 5152), (16, 20, 4096), (11, 4500, 1056), (2, 3, 32), (6, 33, 480)]


@pytest.mark.parametrize("t", [qwhip.F16, qwhip.BF16])
@pytest.mark.parametrize("kind", ["near", "far", "mixed"])
@pytest.mark.parametrize("m,n,k", GEMV_EXACT)
def test_gemv_exact_sums(dev, t, kind, m, n, k):
    """Scales that leave the elements numbers of x's type, scales that do not, both within steps."""
    near, far, mixed = ([120, 121, 122], [100, 101, 102], [111, 114, 117]) if t == qwhip.F16 else ([120, 121, 122], [252, 253, 254], [249, 252, 254])
    scale_bytes = dict(near=near, far=far, mixed=mixed)[kind]
    down = 100 if scale_bytes[-1] > 200 else 0                  # so far down are x and, here, w's values instead of it
    bank = exact_bank(n, k, n + k, scale_bytes)
    x = np.random.default_rng(m).integers(-1, 2, (m, k)).astype(np.float32)
    image, _ = as_type(x * np.float32(2.0 ** -down), t)
    w = (qwmx.values(bank[0], bank[1]) * 2.0 ** -down).astype(np.float32)
    want = exact_product(x, w, 0.5 * 2.0 ** (scale_bytes[0] - 127 - down))
    wv, bufs = put_bank(dev, bank, k)
    _, y32 = gemv(dev, wv, image, t, m, n)
    assert np.array_equal(y32, want)
    free(*bufs)


def form_of(dev, m, n, k, room):
    r = C.c_uint32()
    return dev.lib.qwhip_mxfp4_gemm_form(m, n, k, room, C.byref(r)), r.value


# form, K ranges or not, sizes: odd and even numbers of stages of 256 columns, five to ten of them, that end whole and with one block; rows of
# Y that do and do not leave as 16-byte pieces
GEMM_STEADY = [(f, 0, m, n, k) for f, m, ns in ((0, 3000, (4099, 4104)), (1, 2000, (4099, 4104)), (2, 777, (2501, 2504)), (3, 130, (5001, 5008)), (4, 70, (515, 520)))
               for n, k in zip(ns * 2, (1280, 1312, 2080, 2336))]
GEMM_STEADY += [(0, 1, 1030, 2500, 17440), (1, 1, 500, 4099, 17408), (2, 1, 130, 2003, 5152), (2, 1, 777, 131, 10016), (3, 1, 64, 128, 8224), (3, 1, 260, 1001, 5152), (4, 0, 33, 31, 17440)]


@pytest.mark.parametrize("form,split,m,n,k", GEMM_STEADY)
@pytest.mark.parametrize("t", [qwhip.F32, qwhip.BF16])
def test_gemm_every_form_in_its_steady_loop(dev, form, split, m, n, k, t):
    wb, xb = exact_bank(n, k, n + k, [121, 122, 123]), exact_bank(m, k, m + k + 1, [126, 127])
    need = dev.lib.qwhip_mxfp4_gemm_workspace_bytes(m, n, k) if split else 0
    ran = form_of(dev, m, n, k, need)
    assert ran[0] == form and (ran[1] > 1) == bool(split)
    room = filled(dev, need, 0x7FC00000) if need else None
    want = exact_product(xb[2], wb[2], 0.25 * 2.0 ** (121 + 126 - 254))
    wv, b0 = put_bank(dev, wb, k)
    xv, b1 = put_bank(dev, xb, k)
    got = gemm(dev, wv, xv, m, n, t, workspace=room)
    assert np.array_equal(got, want if t == qwhip.F32 else qo.bf16_bits_to_f32(qo.f32_to_bf16_bits(want)))
    free(*b0, *b1, *([room] if room else []))


FORM_SHAPES = [(0, 0, 3000, 4099, 1312), (1, 0, 2000, 4104, 1312), (2, 0, 777, 2501, 1376), (3, 0, 130, 5001, 1312), (4, 0, 70, 515, 1312), (2, 1, 130, 2003, 5152), (3, 1, 64, 128, 8224)]


@pytest.mark.parametrize("form,split,m,n,k", FORM_SHAPES)
@pytest.mark.parametrize("pad", [3, 8])
def test_gemm_every_form_with_pitches(dev, form, split, m, n, k, pad):
    """Operands inside wider banks, rows of Y apart: what lies between is neither read for the sums nor written."""
    wb, xb = exact_bank(n, k, 5, [122, 123], ld=k + 96), exact_bank(m, k, 6, [126, 127], ld=k + 416)
    wb[1][:, k // 32:], xb[1][:, k // 32:] = 255, 255          # NaN behind every row's end
    need = dev.lib.qwhip_mxfp4_gemm_workspace_bytes(m, n, k) if split else 0
    ran = form_of(dev, m, n, k, need)
    assert ran[0] == form and (ran[1] > 1) == bool(split)
    room = filled(dev, need, 0x7FC00000) if need else None
    want = exact_product(xb[2], wb[2], 0.25 * 2.0 ** (122 + 126 - 254))
    wv, b0 = put_bank(dev, wb, k)
    xv, b1 = put_bank(dev, xb, k)
    assert np.array_equal(gemm(dev, wv, xv, m, n, qwhip.F32, ldy=n + pad, workspace=room), want)
    free(*b0, *b1, *([room] if room else []))


@pytest.mark.parametrize("form,split,m,n,k", FORM_SHAPES)
def test_gemm_every_form_at_the_ends_of_the_scales(dev, form, split, m, n, k):
    """Blocks whose two scales lie at opposite ends (2^127 and 2^-127 among them) and meet in the middle, and blocks that read as NaN: their
    rows and columns are NaN, all others exact."""
    rng = np.random.default_rng(k)
    wb, xb = exact_bank(n, k, 7, [127]), exact_bank(m, k, 8, [127])
    pairs = np.array([(254, 0), (253, 1), (0, 254), (1, 254), (127, 127), (200, 54), (30, 225)])[rng.integers(0, 7, k // 32)]
    wb[1][:], xb[1][:] = pairs[:, 0].astype(np.uint8), pairs[:, 1].astype(np.uint8)
    both = np.repeat(np.exp2(pairs.sum(1) - 254.0), 32).astype(np.float32)
    w, x = wb[2] * both, xb[2]
    rows, cols = [0, m // 2, m - 1], [1, n // 3, n - 1]
    for j, (r, c) in enumerate(zip(rows, cols)):
        at = (0, k // 64, k // 32 - 1)[j]                        # the first block, one in the middle, the last one
        xb[1][r, at], wb[1][c, at] = 255, 255
    nan = np.zeros((m, n), bool)
    nan[rows], nan[:, cols] = True, True
    need = dev.lib.qwhip_mxfp4_gemm_workspace_bytes(m, n, k) if split else 0
    ran = form_of(dev, m, n, k, need)
    assert ran[0] == form and (ran[1] > 1) == bool(split)
    room = filled(dev, need, 0x7FC00000) if need else None
    wv, b0 = put_bank(dev, wb, k)
    xv, b1 = put_bank(dev, xb, k)
    got = gemm(dev, wv, xv, m, n, qwhip.F32, workspace=room)
    assert np.array_equal(np.isnan(got), nan)
    want = exact_product(x, w, 0.25)
    assert np.array_equal(np.where(nan, 0.0, got), np.where(nan, 0.0, want))
    free(*b0, *b1, *([room] if room else []))


@pytest.mark.parametrize("planes", [0, 1, 2, 5, 100])
def test_gemm_takes_no_more_workspace_than_it_is_given(dev, planes):
    m, n, k = 64, 131, 17440
    room_bytes = planes * m * 132 * 4
    wb, xb = exact_bank(n, k, 3, [121, 122]), exact_bank(m, k, 4, [126, 127])
    ran = form_of(dev, m, n, k, room_bytes)
    assert ran[1] <= max(1, planes) and (planes < 5 or ran[1] > 1)
    room = filled(dev, room_bytes + 4096)
    wv, b0 = put_bank(dev, wb, k)
    xv, b1 = put_bank(dev, xb, k)
    y = filled(dev, m * n * 4)
    qwhip.check(dev.lib.qwhip_mxfp4_gemm(dev.stream.handle, C.byref(wv), C.byref(xv), y.ptr, qwhip.F32, 0, room.ptr, room_bytes))
    dev.stream.sync()
    assert np.array_equal(y.download(np.float32, (m, n)), exact_product(xb[2], wb[2], 0.25 * 2.0 ** (121 + 126 - 254)))
    assert (room.download(np.uint8, (room_bytes + 4096,))[room_bytes:] == 0xA5).all()
    free(y, room, *b0, *b1)


@pytest.mark.parametrize("m,n,k", [(64, 128, 8224), (130, 2003, 5152)])
def test_gemm_ranges_captured_on_two_streams(dev, m, n, k):
    """Two graphs of K ranges, each with its own workspace and stream, replayed at once with eager calls between."""
    need = dev.lib.qwhip_mxfp4_gemm_workspace_bytes(m, n, k)
    assert need > 0
    wb, xs = exact_bank(n, k, 8, [121, 122]), [exact_bank(m, k, 9 + i, [126, 127]) for i in range(2)]
    wv, keep = put_bank(dev, wb, k)
    graphs, bufs = [], list(keep)
    for xb in xs:
        st = qwhip.Stream(dev)
        xv, b = put_bank(dev, xb, k)
        y, room = dev.alloc(m * n * 4), filled(dev, need)
        want = exact_product(xb[2], wb[2], 0.25 * 2.0 ** (121 + 126 - 254))
        dev.stream.sync()
        call = lambda st=st, xv=xv, y=y, room=room: qwhip.check(dev.lib.qwhip_mxfp4_gemm(st.handle, C.byref(wv), C.byref(xv), y.ptr, qwhip.F32, 0, room.ptr, need))  # noqa: E731
        graphs.append((qwhip.Graph(st, call), st, y, want, xv))
        bufs += [y, room, *b]
    eager_room = filled(dev, need)
    for _ in range(4):
        for _, _, y, _, _ in graphs:
            qwhip.check(dev.lib.qwhip_fill_u32(dev.stream.handle, y.ptr, 0, m * n))
        dev.stream.sync()
        for g, *_ in graphs:
            g.launch()
        assert np.array_equal(gemm(dev, wv, graphs[0][4], m, n, qwhip.F32, workspace=eager_room), graphs[0][3])
        for _, st, y, want, _ in graphs:
            st.sync()
            assert np.array_equal(y.download(np.float32, (m, n)), want)
    for g, *_ in graphs:
        g.destroy()
    free(eager_room, *bufs)
