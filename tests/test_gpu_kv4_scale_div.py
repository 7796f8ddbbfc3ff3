"""Attention over the 4-bit cache at the ends of what scale_div may be."""
import numpy as np
import pytest

from nimbleml_amd import kernels as K
from oracle import kv4_ref as R
from test_gpu_kv4 import bound, cache_of, normal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("scale", [2e-38, 5e37, 6.2e37, 1.3e38, 3.4e38])
@pytest.mark.parametrize("dk, seq, n", [(64, 1, 100), (128, 3, 700), (32, 1, 5000)])
def test_largest_and_smallest_divisors(gpu, dtype, scale, dk, seq, n):
    """A divisor near the type's ends: scores near zero (an average of all keys), or of some size
    where the queries are as large; the least with queries as small."""
    r = np.random.RandomState(n)
    k, v = normal(r, (1, 2, n, dk), dtype), normal(r, (1, 2, n, dk), dtype)
    q = normal(r, (1, 2, seq, dk), dtype)
    if scale < 1:
        # scores of any size need queries that float16 and three bf16 parts do not hold: zeros
        q[:] = 0
    elif dtype == np.float32:
        q *= np.float32(scale / 64)  # |q·k| below float32's largest at |q| < 20, |k| < 20: few do
        q = np.clip(q, -1e36, 1e36)
    c = cache_of(k, v)
    got = K.kv4_attention(q, c, [n], scale).numpy().astype(np.float64)
    hk, hv = R.held(k), R.held(v)
    scale = float(np.float32(scale))
    want = R.attention(q, hk, hv, [n], None, scale)
    # beside the bound: log2(e) / scale_div is a denormal above 1.23e38, 2^-149 / 2^-128 off at most
    dots = max((np.abs(q[0, j].astype(np.float64)) @ np.abs(hk[0, j]).T).max() for j in range(2)) / scale
    assert np.abs(got - want).max() <= bound(q, hk, hv, scale, dtype) + 2 * dots * 2.0**-21 * np.abs(hv).max()
