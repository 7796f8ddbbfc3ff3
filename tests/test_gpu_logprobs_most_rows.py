"""The most rows that a call takes, 2^31 − 1 (of one logit and of two): the last launches' rows are
their own, and the calls end."""
import numpy as np
import pytest

from nimbleml_amd import _native as N

pytestmark = pytest.mark.gpu

ROWS = 2**31 - 1
SEAMS = [0, 2**21 - 3, 2**31 - 2**21 - 3, ROWS - 6]  # six rows from each are looked at
FILL = 0x3C  # every byte: 1.0586 in float16, 0.0115 in float32


def array(n, dtype, byte=FILL):
    a = N.DeviceArray((n,), dtype)
    N.check(N.lib.nml_memset(a.ptr, byte, a.nbytes))
    return a


def put(a, at, values):
    v = np.ascontiguousarray(values, a.dtype)
    N.check(N.lib.nml_memcpy_h2d(a.ptr + at * v.itemsize, v.ctypes.data, v.nbytes))


def get(a, at, n):
    v = np.empty(n, a.dtype)
    N.check(N.lib.nml_memcpy_d2h(v.ctypes.data, a.ptr + at * v.itemsize, v.nbytes))
    return v


def test_most_rows_of_statistics(gpu):
    x, m = array(ROWS, np.float16), array(ROWS, np.float32, 0xFF)
    r = np.random.RandomState(1)
    for at in SEAMS:
        put(x, at, r.randn(6))
    N.check(N.lib.nml_token_logprobs_device(x.ptr, 1, None, ROWS, 1, 0, 0, 0, None, None, m.ptr, None,
                                            None, None, None, N.F16))
    for at in SEAMS + [2**30, ROWS // 3]:  # a row's largest logit is its only one
        assert np.array_equal(get(m, at, 6), get(x, at, 6).astype(np.float32)), at


def test_most_rows_of_the_gradient(gpu):
    x, d = array(2 * ROWS, np.float16), array(2 * ROWS, np.float16, 0xFF)
    t, s = array(ROWS, np.int64, 0), array(ROWS, np.float32)  # s: m, l and dlogp of most rows
    r = np.random.RandomState(2)
    for at in SEAMS:
        put(x, 2 * at, r.randn(12))
        put(t, at, [0, 1, 1, 0, 1, 0])
    N.check(N.lib.nml_token_logprobs_backward_device(
        x.ptr, 2, t.ptr, s.ptr, s.ptr, None, s.ptr, None, ROWS, 2, 0, 0, d.ptr, 2, None, N.F16))
    c = get(s, 0, 1).astype(np.float64)[0]
    for at in SEAMS + [2**30, ROWS // 3]:
        lg, hot = get(x, 2 * at, 12).reshape(6, 2).astype(np.float64), get(t, at, 6)[:, None] == np.arange(2)
        want = c * (hot - np.exp(lg - c - np.log(c)))
        # |log p| < 8: p to 12·2^-22 relative, then half a step of float16, or half of its least value
        tol = np.abs(want) * 2.0**-11 + 2.0**-25 + c * np.exp(lg - c - np.log(c)) * 12 * 2.0**-22
        assert (np.abs(get(d, 2 * at, 12).reshape(6, 2) - want) <= tol).all(), at
