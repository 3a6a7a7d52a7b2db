"""qwhip_mxfp4_gemm_form and _workspace_bytes agree, on a host without a GPU."""
import ctypes as C

import pytest

from qwegn_amd import qwhip

ROWS_FORM = 4


@pytest.fixture(scope="module")
def lib():
    return qwhip.load()


def form(lib, m, n, k, room):
    r = C.c_uint32(77)
    return lib.qwhip_mxfp4_gemm_form(m, n, k, room, C.byref(r)), r.value


def test_nothing_to_multiply(lib):
    for m, n, k in ((0, 8, 32), (8, 0, 32), (8, 8, 0), (8, 8, 48)):
        assert form(lib, m, n, k, 1 << 40) == (ROWS_FORM, 1)
        assert lib.qwhip_mxfp4_gemm_workspace_bytes(m, n, k) == 0
    assert lib.qwhip_mxfp4_gemm_form(8, 8, 32, 0, None) == ROWS_FORM


@pytest.mark.parametrize("m", [1, 63, 64, 128, 200, 777, 4096])
@pytest.mark.parametrize("n", [1, 127, 128, 1003, 5120])
@pytest.mark.parametrize("k", [32, 1312, 9632, 17408])
def test_the_room_that_is_asked_for_is_the_room_that_is_used(lib, m, n, k):
    need = lib.qwhip_mxfp4_gemm_workspace_bytes(m, n, k)
    best = form(lib, m, n, k, 1 << 60)
    planes = m * ((n + 3) // 4 * 4) * 4
    assert need == (best[1] * planes if best[1] > 1 else 0)
    assert form(lib, m, n, k, need) == best
    assert form(lib, m, n, k, 0)[1] == 1
    if need:
        assert form(lib, m, n, k, need - 1)[1] < best[1] or form(lib, m, n, k, need - 1) != best
    if m < 64 or n < 128:
        assert best[0] == ROWS_FORM
