"""MXFP4 products where they can go wrong: scales at the ends of their range, operands of very many rows, every kernel form in its steady loop,
and data whose sums fp32 holds exactly, so that one element out of a long row shows."""
import ctypes as C

import numpy as np
import pytest

from oracle import qwmx
from qwegn_amd import qwhip
from tests.test_gpu_mxfp4 import as_type, check_product, free, gemm, gemv, put_bank, random_bank

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
