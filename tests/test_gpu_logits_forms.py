"""qwhip_logits_process where a row's slices, ties and zeros can go wrong, against the rules in numpy (oracle/qwmx.py), bit for bit."""
import ctypes as C

import numpy as np
import pytest

from oracle import qwmx
from oracle import qworacle as qo
from qwegn_amd import qwhip
from tests.test_gpu_logits import Step, equal, image_of, rounded, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return qwhip.Device(0)


@pytest.mark.parametrize("t", [qwhip.F32, qwhip.F16, qwhip.BF16])
@pytest.mark.parametrize("rows,n", [(3, 9), (1, 40000), (130, 16384), (256, 32003)])
def test_zeros_of_both_signs(dev, t, rows, n):
    """A row whose largest result is a zero: +0 is above -0, as the fold of qwhip_argmax_f32 has it, then the lower token wins."""
    rng = np.random.default_rng(n)
    x = -np.abs(rng.standard_normal((rows, n))) - 0.01
    for r in range(rows):
        low, high = np.sort(rng.choice(n, 2, replace=False))
        x[r, low], x[r, high] = ((-0.0, 0.0), (0.0, -0.0), (-0.0, -0.0), (0.0, 0.0))[r % 4]
    if n > 2048:
        x[rows - 1] = -1.0
        x[rows - 1, [7, 7 + 1024, 9]] = -0.0, 0.0, -0.0      # one thread's own where it has several
    image, val = image_of(x, t)
    assert (np.signbit(val) | (val == 0)).all()
    step = Step(dev, rows, n)
    want, tokens = qwmx.logits_f32(val)
    assert np.array_equal(tokens, qo.head_argmax(val))
    got, tok = run(dev, step, image, t)
    assert equal(got, rounded(want, t))
    assert np.array_equal(tok, tokens)
    src, out = dev.put(val), dev.alloc(rows * 4)
    qwhip.check(dev.lib.qwhip_argmax_f32(dev.stream.handle, src.ptr, rows, n, out.ptr))
    dev.stream.sync()
    assert np.array_equal(out.download(np.int32, (rows,)), tokens)
    src.free()
    out.free()
