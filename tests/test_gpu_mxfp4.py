"""MXFP4 through the C ABI against the definitions in 64 bits (oracle/qwmx.py).

Quantiser and dequant: equal, bit for bit.  Products: the operands' values are exact and so is a product of two of them in fp32, which
leaves the sums: k additions, each off by at most one step of its result (2^-23; a rounding is half of that, a matrix unit that truncates
the whole), so |error| <= (k + 32) 2^-23 sum |x w|, and half a step of the output's type at the store."""
import ctypes as C

import numpy as np
import pytest

from oracle import qwmx
from oracle import qworacle as qo
from qwegn_amd import qwhip

pytestmark = pytest.mark.gpu
HALF = {qwhip.F32: 2.0 ** -24, qwhip.F16: 2.0 ** -11, qwhip.BF16: 2.0 ** -8}
LEAST = {qwhip.F32: 2.0 ** -126, qwhip.F16: 2.0 ** -24, qwhip.BF16: 2.0 ** -126}   # half a step of the subnormals and then some
SIZE = {qwhip.F32: 4, qwhip.F16: 2, qwhip.BF16: 2}


@pytest.fixture(scope="module")
def dev():
    return qwhip.Device(0)


def as_type(x, t):
    """(device image, the values it stands for as f32)"""
    with np.errstate(over="ignore", invalid="ignore"):
        if t == qwhip.F32:
            return x.astype(np.float32), x.astype(np.float32)
        if t == qwhip.F16:
            h = x.astype(np.float16)
            return h, h.astype(np.float32)
        b = qo.f32_to_bf16_bits(x.astype(np.float32))
        return b, qo.bf16_bits_to_f32(b)


def read(buf, t, shape, stream=None):
    raw = buf.download(qwhip.NP_DTYPES[t], shape, stream)
    return qo.bf16_bits_to_f32(raw) if t == qwhip.BF16 else raw.astype(np.float32)


def filled(dev, nbytes, word=0xA5A5A5A5):
    buf = dev.alloc((nbytes + 259) // 4 * 4)
    qwhip.check(dev.lib.qwhip_fill_u32(dev.stream.handle, buf.ptr, word, buf.nbytes // 4))
    return buf


def view(codes, scales, n, k, ld=0):
    return qwhip.Mxfp4View(codes.ptr, scales.ptr, codes.nbytes, scales.nbytes, n, k, ld)


def random_bank(n, k, seed, spread=4, ld=None):
    """Codes and scale bytes drawn as such (every code, scales over 2^spread either side of 2^-6), rows `ld` apart with other bytes between."""
    rng = np.random.default_rng(seed)
    ld = ld or k
    codes = rng.integers(0, 256, (n, ld // 2), dtype=np.uint8)
    scales = rng.integers(121 - spread, 122 + spread, (n, ld // 32)).astype(np.uint8)
    return codes, scales, qwmx.values(codes[:, :k // 2], scales[:, :k // 32])


def put_bank(dev, bank, k):
    codes, scales, _ = bank
    n, ld = codes.shape[0], codes.shape[1] * 2
    cb, sb = dev.put(codes), dev.put(scales)
    return view(cb, sb, n, k, 0 if ld == k else ld), (cb, sb)


def check_product(got, x, w, t):
    ref = x @ w.T
    bound = (x.shape[1] + 32) * 2.0 ** -23 * (np.abs(x) @ np.abs(w).T)
    bound = bound + HALF[t] * (np.abs(ref) + bound) + LEAST[t]
    worst = np.max(np.abs(got - ref) / bound)
    assert worst <= 1.0, f"{worst} of the bound"


def free(*bufs):
    for b in bufs:
        b.free()


# ---- quantiser ---------------------------------------------------------------------------------------------------------------------
def quantise(dev, x, t, ld=None, with_values=True):
    image, val = as_type(x, t)
    rows, k = image.shape
    ld = ld or k
    wide = np.full((rows, ld), 0x4242, image.dtype)
    wide[:, :k] = image
    src = dev.put(wide)
    codes, scales, values = filled(dev, rows * k // 2), filled(dev, rows * k // 32), filled(dev, rows * k * SIZE[t])
    qwhip.check(dev.lib.qwhip_quantize_mxfp4(dev.stream.handle, src.ptr, t, rows, k, 0 if ld == k else ld, codes.ptr, scales.ptr, values.ptr if with_values else None))
    c, s, v = codes.download(np.uint8, (rows, k // 2)), scales.download(np.uint8, (rows, k // 32)), read(values, t, (rows, k))
    tails = [b.download(np.uint8, (b.nbytes,))[used:used + 256] for b, used in ((codes, rows * k // 2), (scales, rows * k // 32), (values, rows * k * SIZE[t]))]
    for tail, name in zip(tails, ("codes", "scales", "values")):
        assert (tail[: len(tail) // 4 * 4] == 0xA5).all(), f"{name}: written behind the end"
    free(src, codes, scales, values)
    return c, s, v, val


def check_quantised(c, s, v, val, with_values=True):
    want_c, want_s = qwmx.quantise(val)
    assert np.array_equal(s, want_s)
    assert np.array_equal(c, want_c)
    if with_values:
        assert np.array_equal(v.astype(np.float64), qwmx.values(want_c, want_s), equal_nan=True)


@pytest.mark.parametrize("t", [qwhip.F32, qwhip.F16, qwhip.BF16])
@pytest.mark.parametrize("rows,k,ld", [(1, 32, None), (1, 5120, None), (3, 96, 128), (65, 1056, None), (7, 2080, 2112), (33, 32, 40), (2, 17408, None)])
def test_quantise_rows(dev, t, rows, k, ld):
    rng = np.random.default_rng(rows * k)
    x = rng.standard_normal((rows, k)) * np.exp2(rng.integers(-6, 6, (rows, 1)))
    x[rng.random((rows, k)) < 0.01] *= 20.0
    check_quantised(*quantise(dev, x, t, ld))


def test_quantise_without_values(dev):
    x = np.random.default_rng(0).standard_normal((5, 160))
    c, s, v, val = quantise(dev, x, qwhip.BF16, with_values=False)
    check_quantised(c, s, v, val, with_values=False)
    assert np.array_equal(v, np.full_like(v, qo.bf16_bits_to_f32(np.array([0xA5A5], np.uint16))[0]))


@pytest.mark.parametrize("t", [qwhip.F32, qwhip.F16, qwhip.BF16])
def test_quantise_borders_and_odd_values(dev, t):
    """Every border between two elements and its neighbours under scales from the smallest to the largest of the type, zeros of both signs,
    blocks of zeros, of subnormals, with an infinity, with a NaN."""
    near = np.concatenate([[b, b * (1 - 2.0 ** -7), b * (1 + 2.0 ** -7)] for b in np.append(qwmx.BORDERS, [5.0, 6.0, 7.0])])          # thirty of them
    low, high = {qwhip.F32: (-140, 125), qwhip.F16: (-20, 13), qwhip.BF16: (-130, 125)}[t]
    rows = []
    for e in range(low, high + 1, 3):
        for sign in (1.0, -1.0):
            rows.append(np.concatenate([near, [4.0, 7.5]]) * sign * 2.0 ** e)
    tiny = {qwhip.F32: 2.0 ** -149, qwhip.F16: 2.0 ** -24, qwhip.BF16: 2.0 ** -133}[t]
    odd = [np.zeros(32), -np.zeros(32), np.full(32, tiny), np.arange(-16, 16) * tiny, np.full(32, np.inf), np.full(32, np.nan)]
    for bad in (np.inf, -np.inf, np.nan):
        for at in (0, 13, 31):
            v = np.arange(32.0)
            v[at] = bad
            odd.append(v)
    biggest = {qwhip.F32: np.finfo(np.float32).max, qwhip.F16: 65504.0, qwhip.BF16: 2.0 ** 127 * 1.9921875}[t]
    odd += [np.full(32, biggest), np.linspace(-1, 1, 32) * biggest]
    check_quantised(*quantise(dev, np.stack(rows + odd), t))


def test_quantise_every_bf16(dev):
    """All 65,536 bf16 numbers, in blocks of neighbours and in blocks of a random order."""
    bits = np.arange(65536, dtype=np.uint16)
    for order in (bits, np.random.default_rng(5).permutation(bits)):
        check_quantised(*quantise(dev, qo.bf16_bits_to_f32(order).reshape(-1, 64), qwhip.BF16))


# ---- dequant -----------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("t", [qwhip.F32, qwhip.F16, qwhip.BF16])
def test_dequant_every_code_under_every_scale(dev, t):
    codes = np.tile(np.array([(2 * i % 16) | ((2 * i + 1) % 16) << 4 for i in range(16)], np.uint8), (256, 1))
    scales = np.arange(256, dtype=np.uint8).reshape(256, 1)
    v, bufs = put_bank(dev, (codes, scales, None), 32)
    out = filled(dev, 256 * 32 * SIZE[t])
    qwhip.check(dev.lib.qwhip_dequant_mxfp4(dev.stream.handle, C.byref(v), out.ptr, t))
    got = read(out, t, (256, 32)).astype(np.float64)
    want = qwmx.values(codes, scales)
    want = np.where(np.abs(want) >= 2.0 ** 128, np.copysign(np.inf, want), want)   # 4 x 2^126 and on: over fp32 and bf16
    with np.errstate(over="ignore", invalid="ignore"):
        want = want.astype(np.float16).astype(np.float64) if t == qwhip.F16 else want
    assert np.array_equal(got, want, equal_nan=True)
    free(out, *bufs)


@pytest.mark.parametrize("n,k,ld", [(1, 32, 64), (5, 96, 96), (9, 160, 224)])
def test_dequant_pitch(dev, n, k, ld):
    bank = random_bank(n, k, 3, ld=ld)
    v, bufs = put_bank(dev, bank, k)
    out = dev.alloc(n * k * 4)
    qwhip.check(dev.lib.qwhip_dequant_mxfp4(dev.stream.handle, C.byref(v), out.ptr, qwhip.F32))
    assert np.array_equal(read(out, qwhip.F32, (n, k)).astype(np.float64), bank[2])
    free(out, *bufs)


# ---- product of two quantised operands ---------------------------------------------------------------------------------------------
def gemm(dev, wv, xv, m, n, t, ldy=0, workspace=None, stream=None):
    pitch = ldy or n
    y = filled(dev, m * pitch * SIZE[t])
    dev.stream.sync()
    st = (stream or dev.stream).handle
    qwhip.check(dev.lib.qwhip_mxfp4_gemm(st, C.byref(wv), C.byref(xv), y.ptr, t, ldy, workspace.ptr if workspace else None, workspace.nbytes if workspace else 0))
    raw = y.download(qwhip.NP_DTYPES[t], (m * pitch + 64,), stream)
    mark = np.frombuffer(b"\xA5" * 4, qwhip.NP_DTYPES[t])[0]
    assert (raw[m * pitch:].view(np.uint8) == 0xA5).all(), "written behind the last row"
    body = raw[: m * pitch].reshape(m, pitch)
    assert (body[:, n:] == mark).all(), "written between the rows"
    body = np.ascontiguousarray(body[:, :n])
    y.free()
    return qo.bf16_bits_to_f32(body) if t == qwhip.BF16 else body.astype(np.float32)


GEMM_SHAPES = [(1, 1, 32), (1, 640, 1024), (16, 640, 1024), (3, 17, 64), (77, 1003, 1056), (64, 256, 128), (129, 130, 160), (255, 257, 96), (257, 511, 1312), (256, 256, 5120),
               (512, 768, 512), (300, 4099, 288), (33, 48, 17408), (1000, 320, 2080), (700, 1028, 544), (513, 1030, 768), (260, 516, 2048), (2, 5120, 640), (40, 2560, 992),
               # whole and half tiles, edges that overlap, K ranges (with a workspace), columns that end inside a stage
               (64, 128, 32), (70, 200, 96), (1000, 1000, 1024), (2048, 5100, 288), (6000, 5000, 96), (200, 650, 17408), (520, 517, 9632), (8026, 300, 64)]


@pytest.mark.parametrize("m,n,k", GEMM_SHAPES)
@pytest.mark.parametrize("t,ws", [(qwhip.F32, 0), (qwhip.F32, 1), (qwhip.F16, 1), (qwhip.BF16, 0)])
def test_gemm(dev, m, n, k, t, ws):
    wb, xb = random_bank(n, k, n + k), random_bank(m, k, m + k + 1)
    wv, b0 = put_bank(dev, wb, k)
    xv, b1 = put_bank(dev, xb, k)
    need = dev.lib.qwhip_mxfp4_gemm_workspace_bytes(m, n, k)
    room = filled(dev, need, 0x7FC00000) if ws else None      # what was in the workspace before does not count
    check_product(gemm(dev, wv, xv, m, n, t, workspace=room), xb[2], wb[2], t)
    free(*b0, *b1, *([room] if ws else []))


@pytest.mark.parametrize("m,n,k,ldw,ldx,ldy", [(70, 300, 160, 192, 480, 311), (300, 520, 640, 672, 704, 520), (17, 33, 32, 64, 32, 40), (515, 260, 512, 512, 576, 264)])
@pytest.mark.parametrize("t", [qwhip.F32, qwhip.BF16])
def test_gemm_pitches(dev, m, n, k, ldw, ldx, ldy, t):
    wb, xb = random_bank(n, k, 1, ld=ldw), random_bank(m, k, 2, ld=ldx)
    wv, b0 = put_bank(dev, wb, k)
    xv, b1 = put_bank(dev, xb, k)
    check_product(gemm(dev, wv, xv, m, n, t, ldy=ldy), xb[2], wb[2], t)
    free(*b0, *b1)


@pytest.mark.parametrize("m,n,k", [(37, 50, 96), (300, 270, 384)])
def test_gemm_scales_out_of_reach(dev, m, n, k):
    """Operands whose scales lie far apart (the product does not), and blocks that read as NaN: exactly their rows and columns are NaN."""
    wb, xb = random_bank(n, k, 3), random_bank(m, k, 4)
    ws, xs = wb[1].astype(int) - 100, xb[1].astype(int) + 100
    ws[:, 1] = 0                                              # 2^-127: nothing of it shows beside the others
    ws, xs = ws.astype(np.uint8), xs.astype(np.uint8)
    ws[7, 0] = 255
    xs[5, 2] = 255
    w, x = qwmx.values(wb[0], ws), qwmx.values(xb[0], xs)
    wv, b0 = put_bank(dev, (wb[0], ws, None), k)
    xv, b1 = put_bank(dev, (xb[0], xs, None), k)
    got = gemm(dev, wv, xv, m, n, qwhip.F32)
    nan = np.zeros((m, n), bool)
    nan[5], nan[:, 7] = True, True
    assert np.array_equal(np.isnan(got), nan)
    w[7], x[5] = 0.0, 0.0
    check_product(np.where(nan, 0.0, got), x, w, qwhip.F32)
    free(*b0, *b1)


def test_gemm_captured_and_on_two_streams(dev):
    """Two graphs, each with its own workspace and stream, replayed in turn with eager calls between: the eager bits every time."""
    m, n, k = 24, 640, 4096
    wb, xs = random_bank(n, k, 8), [random_bank(m, k, 9 + i) for i in range(2)]
    wv, keep = put_bank(dev, wb, k)
    need = dev.lib.qwhip_mxfp4_gemm_workspace_bytes(m, n, k)
    eager, graphs, outs, rooms = [], [], [], []
    for i in range(2):
        st = qwhip.Stream(dev)
        xv, b = put_bank(dev, xs[i], k)
        y, room = dev.alloc(m * n * 4), filled(dev, need)
        dev.stream.sync()
        eager.append(gemm(dev, wv, xv, m, n, qwhip.F32, workspace=room))
        call = lambda st=st, xv=xv, y=y, room=room: qwhip.check(dev.lib.qwhip_mxfp4_gemm(st.handle, C.byref(wv), C.byref(xv), y.ptr, qwhip.F32, 0, room.ptr, room.nbytes))  # noqa: E731
        graphs.append((qwhip.Graph(st, call), st))
        outs.append(y)
        rooms.append((room, b))
    for _ in range(4):
        for y in outs:
            qwhip.check(dev.lib.qwhip_fill_u32(dev.stream.handle, y.ptr, 0, m * n))
        dev.stream.sync()
        for g, _st in graphs:
            g.launch()
        for (_, st), y, want in zip(graphs, outs, eager):
            st.sync()
            assert np.array_equal(y.download(np.float32, (m, n)), want)
    for g, _st in graphs:
        g.destroy()
    check_product(eager[0], xs[0][2], wb[2], qwhip.F32)
    free(*keep, *outs, *[r for r, _ in rooms])


# ---- 16-bit rows with quantised weights ----------------------------------------------------------------------------------------------
def gemv(dev, wv, x_image, t, m, n, both=False, half=False):
    xb = dev.put(x_image)
    y16, y32 = filled(dev, m * n * 2), filled(dev, m * n * 4)
    qwhip.check(dev.lib.qwhip_mxfp4_gemv(dev.stream.handle, C.byref(wv), xb.ptr, t, m, y16.ptr if half or both else None, None if half else y32.ptr))
    a, b = y16.download(np.uint8, (m * n * 2 + 64,)), y32.download(np.uint8, (m * n * 4 + 64,))
    assert (a[m * n * 2:] == 0xA5).all() and (b[m * n * 4:] == 0xA5).all(), "written behind the last row"
    free(xb, y16, y32)
    return a[: m * n * 2].view(np.float16).reshape(m, n).astype(np.float32), b[: m * n * 4].view(np.float32).reshape(m, n)


@pytest.mark.parametrize("m", [1, 2, 3, 5, 8, 13, 16])
@pytest.mark.parametrize("n,k,ld", [(1, 32, None), (640, 1024, None), (17, 96, 128), (1003, 1056, None), (333, 2080, 2112), (96, 17408, None), (4100, 288, None), (31, 5120, None)])
@pytest.mark.parametrize("t", [qwhip.F16, qwhip.BF16])
def test_gemv(dev, m, n, k, ld, t):
    bank = random_bank(n, k, n, ld=ld)
    wv, bufs = put_bank(dev, bank, k)
    image, val = as_type(np.random.default_rng(m).standard_normal((m, k)), t)
    y16, y32 = gemv(dev, wv, image, t, m, n, both=True)
    check_product(y32, val.astype(np.float64), bank[2], qwhip.F32)
    check_product(y16, val.astype(np.float64), bank[2], qwhip.F16)
    only, _ = gemv(dev, wv, image, t, m, n, half=True)
    assert np.array_equal(only, y16)
    free(*bufs)


@pytest.mark.parametrize("t", [qwhip.F16, qwhip.BF16])
@pytest.mark.parametrize("m,n,k", [(1, 40007, 64), (4, 17001, 544), (7, 9000, 2592), (16, 4500, 1056), (3, 5000, 3616), (2, 35, 33312), (1, 20, 90112), (9, 333, 17408), (11, 2116, 8768), (16, 4200, 8224)])
def test_gemv_workgroups_with_several_tiles_and_long_rows(dev, t, m, n, k):
    bank = random_bank(n, k, n)
    wv, bufs = put_bank(dev, bank, k)
    image, val = as_type(np.random.default_rng(m).standard_normal((m, k)), t)
    _, y32 = gemv(dev, wv, image, t, m, n)
    check_product(y32, val.astype(np.float64), bank[2], qwhip.F32)
    free(*bufs)


@pytest.mark.parametrize("t", [qwhip.F16, qwhip.BF16])
@pytest.mark.parametrize("m", [1, 6])
def test_gemv_scales_out_of_reach(dev, t, m):
    """Weights far outside f16's range meet small activations; NaN blocks show in their rows alone, also beside the end of a row."""
    n, k = 40, 160
    bank = random_bank(n, k, 5)
    scales = bank[1].astype(int) + 30
    scales[:, 3] = 0
    scales = scales.astype(np.uint8)
    scales[9, 4], scales[10, 0] = 255, 255
    image, val = as_type(np.random.default_rng(m).standard_normal((m, k)) * 2.0 ** -10, t)
    wv, bufs = put_bank(dev, (bank[0], scales, None), k)
    _, y32 = gemv(dev, wv, image, t, m, n)
    w = qwmx.values(bank[0], scales)
    assert np.array_equal(np.isnan(y32), np.isnan(val.astype(np.float64) @ w.T))
    w[[9, 10]] = 0.0
    check_product(np.where(np.isnan(y32), 0.0, y32), val.astype(np.float64), w, qwhip.F32)
    free(*bufs)


@pytest.mark.parametrize("t", [qwhip.F16, qwhip.BF16])
@pytest.mark.parametrize("byte", [0, 1, 2, 250, 252])
def test_gemv_scales_at_the_ends(dev, t, byte):
    """Every scale the smallest or the largest there is, with activations that bring the results back among fp32's normal numbers."""
    n, k = 33, 672
    bank = random_bank(n, k, 9)
    scales = np.full_like(bank[1], byte)
    image, val = as_type(np.random.default_rng(2).standard_normal((2, k)) * (2.0 ** 14 if byte < 100 else 2.0 ** -14), t)
    wv, bufs = put_bank(dev, (bank[0], scales, None), k)
    _, y32 = gemv(dev, wv, image, t, 2, n)
    w, x = qwmx.values(bank[0], scales), val.astype(np.float64)
    # a term under 2^-126 may lose what lies under 2^-149, half a step of fp32's subnormals, k of them
    bound = (k + 32) * 2.0 ** -23 * (np.abs(x) @ np.abs(w).T) + k * 2.0 ** -149
    assert (np.abs(y32 - x @ w.T) <= bound).all()
    free(*bufs)


@pytest.mark.parametrize("t", [qwhip.F16, qwhip.BF16])
@pytest.mark.parametrize("byte", [113, 114, 140, 141])
def test_gemv_scales_about_the_normal_f16_numbers(dev, t, byte):
    """Scales whose elements begin or cease to be normal f16 numbers, alone and mixed with others inside steps, rows and waves."""
    n, k = 50, 2336
    bank = random_bank(n, k, 19)
    scales = np.full_like(bank[1], byte)
    scales[17:30, ::5] = 121
    scales[30:, 40:] = 127
    scales[40, 3] = 90
    image, val = as_type(np.random.default_rng(3).standard_normal((3, k)), t)
    wv, bufs = put_bank(dev, (bank[0], scales, None), k)
    _, y32 = gemv(dev, wv, image, t, 3, n)
    check_product(y32, val.astype(np.float64), qwmx.values(bank[0], scales), qwhip.F32)
    free(*bufs)


@pytest.mark.parametrize("m,n,k", [(1, 700, 1056), (5, 333, 2592), (16, 96, 17408), (8, 200, 9216)])
def test_gemv_f16_scales_in_and_out_of_range(dev, m, n, k):
    bank = random_bank(n, k, m, spread=9)                       # 2^-15 .. 2^3: some steps of a wave are in range, some are not
    bank[1][: n // 2] = np.maximum(bank[1][: n // 2], 114)
    w = qwmx.values(bank[0], bank[1])
    wv, bufs = put_bank(dev, bank, k)
    image, val = as_type(np.random.default_rng(m).standard_normal((m, k)), qwhip.F16)
    _, y32 = gemv(dev, wv, image, qwhip.F16, m, n)
    check_product(y32, val.astype(np.float64), w, qwhip.F32)
    free(*bufs)


@pytest.mark.parametrize("t", [qwhip.F16, qwhip.BF16])
def test_gemv_small_activations(dev, t):
    """Activations among the subnormal numbers of f16."""
    n, k, m = 64, 1120, 4
    bank = random_bank(n, k, 23)
    image, val = as_type(np.random.default_rng(4).standard_normal((m, k)) * 2.0 ** -17, t)
    wv, bufs = put_bank(dev, bank, k)
    _, y32 = gemv(dev, wv, image, t, m, n)
    check_product(y32, val.astype(np.float64), bank[2], qwhip.F32)
    free(*bufs)


def test_gemv_captured(dev):
    n, k, m = 640, 2048, 3
    bank = random_bank(n, k, 6)
    wv, bufs = put_bank(dev, bank, k)
    image, _ = as_type(np.random.default_rng(1).standard_normal((m, k)), qwhip.F16)
    _, want = gemv(dev, wv, image, qwhip.F16, m, n)
    xb, y = dev.put(image), dev.alloc(m * n * 4)
    g = qwhip.Graph(dev.stream, lambda: qwhip.check(dev.lib.qwhip_mxfp4_gemv(dev.stream.handle, C.byref(wv), xb.ptr, qwhip.F16, m, None, y.ptr)))
    for _ in range(3):
        qwhip.check(dev.lib.qwhip_fill_u32(dev.stream.handle, y.ptr, 0, m * n))
        g.launch()
        dev.stream.sync()
        assert np.array_equal(y.download(np.float32, (m, n)), want)
    g.destroy()
    free(xb, y, *bufs)


@pytest.mark.parametrize("m,n,k", [(512, 640, 8192), (300, 4000, 640), (2048, 5100, 288)])
def test_gemm_forms_captured(dev, m, n, k):
    """The tiled kernel, with K ranges where there is room for them, recorded and replayed: the eager bits."""
    wb, xb = random_bank(n, k, 1), random_bank(m, k, 2)
    wv, b0 = put_bank(dev, wb, k)
    xv, b1 = put_bank(dev, xb, k)
    room = filled(dev, dev.lib.qwhip_mxfp4_gemm_workspace_bytes(m, n, k), 0x7FC00000)
    want = gemm(dev, wv, xv, m, n, qwhip.F32, workspace=room)
    y, st = dev.alloc(m * n * 4), qwhip.Stream(dev)
    g = qwhip.Graph(st, lambda: qwhip.check(dev.lib.qwhip_mxfp4_gemm(st.handle, C.byref(wv), C.byref(xv), y.ptr, qwhip.F32, 0, room.ptr, room.nbytes)))
    for _ in range(3):
        qwhip.check(dev.lib.qwhip_fill_u32(dev.stream.handle, y.ptr, 0, m * n))
        qwhip.check(dev.lib.qwhip_fill_u32(dev.stream.handle, room.ptr, 0x7FC00000, room.nbytes // 4))
        dev.stream.sync()
        g.launch()
        st.sync()
        assert np.array_equal(y.download(np.float32, (m, n)), want)
    g.destroy()
    check_product(want, xb[2], wb[2], qwhip.F32)
    free(y, room, *b0, *b1)


@pytest.mark.parametrize("m,n,k", [(8, 200, 17408), (13, 640, 12800), (2, 96, 17408)])
def test_gemv_with_much_lds_captured(dev, m, n, k):
    bank = random_bank(n, k, 6)
    wv, bufs = put_bank(dev, bank, k)
    image, val = as_type(np.random.default_rng(1).standard_normal((m, k)), qwhip.BF16)
    xb, y, st = dev.put(image), dev.alloc(m * n * 4), qwhip.Stream(dev)
    g = qwhip.Graph(st, lambda: qwhip.check(dev.lib.qwhip_mxfp4_gemv(st.handle, C.byref(wv), xb.ptr, qwhip.BF16, m, None, y.ptr)))
    _, want = gemv(dev, wv, image, qwhip.BF16, m, n)
    for _ in range(3):
        qwhip.check(dev.lib.qwhip_fill_u32(dev.stream.handle, y.ptr, 0, m * n))
        dev.stream.sync()
        g.launch()
        st.sync()
        assert np.array_equal(y.download(np.float32, (m, n)), want)
    g.destroy()
    check_product(want, val.astype(np.float64), bank[2], qwhip.F32)
    free(xb, y, *bufs)


def test_quantise_and_dequant_captured(dev):
    rows, k = 33, 1056
    x = np.random.default_rng(7).standard_normal((rows, k)).astype(np.float32)
    src, codes, scales, values, out = dev.put(x), dev.alloc(rows * k // 2), dev.alloc(rows * k // 32), dev.alloc(rows * k * 4), dev.alloc(rows * k * 4)
    v, st = view(codes, scales, rows, k), qwhip.Stream(dev)

    def both():
        qwhip.check(dev.lib.qwhip_quantize_mxfp4(st.handle, src.ptr, qwhip.F32, rows, k, 0, codes.ptr, scales.ptr, values.ptr))
        qwhip.check(dev.lib.qwhip_dequant_mxfp4(st.handle, C.byref(v), out.ptr, qwhip.F32))

    g = qwhip.Graph(st, both)
    for turn in range(3):
        x = np.random.default_rng(turn).standard_normal((rows, k)).astype(np.float32)
        src.upload(x)
        g.launch()
        st.sync()
        want = qwmx.values(*qwmx.quantise(x))
        assert np.array_equal(values.download(np.float32, (rows, k)).astype(np.float64), want)
        assert np.array_equal(out.download(np.float32, (rows, k)).astype(np.float64), want)
    g.destroy()
    free(src, codes, scales, values, out)
