"""Values near float32's largest in the 4-bit cache: their weighted average is finite as they are."""
import numpy as np
import pytest

from nimbleml_amd import kernels as K
from oracle import kv4_ref as R
from test_gpu_kv4 import cache_of, normal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dk, group, seq", [(64, 1, 1), (64, 2, 3), (96, 1, 1), (256, 1, 2)])
@pytest.mark.parametrize("lens", [[1, 2, 3, 33], [40, 700, 300, 1], [5000, 3, 129, 4097]])
def test_averages_of_the_largest_values(gpu, dk, group, seq, lens):
    """Block 0 of V near 2.5e38 of one sign, block 1 of both signs, the rest ordinary; with one block
    of 1e-30 the other way: each block's error is relative to its own values."""
    r = np.random.RandomState(dk + seq)
    b, p = len(lens), max(lens)
    k = normal(r, (b, 1, p, dk), np.float32)
    v = normal(r, (b, 1, p, dk), np.float32)
    v[..., :32] = r.uniform(1e38, 3.4e38, v[..., :32].shape)
    v[..., 32:64] = r.uniform(1e38, 3.4e38, v[..., :32].shape) * r.choice([-1, 1], v[..., :32].shape)
    v[1, ..., :32] = 1e-30 * r.randn(*v[1, ..., :32].shape)
    v = v.astype(np.float32)
    q = normal(r, (b, group, seq, dk), np.float32)
    scale = float(np.sqrt(dk))
    got = K.kv4_attention(q, cache_of(k, v), lens, scale).numpy().astype(np.float64)
    hk, hv = R.held(k), R.held(v)
    want = R.attention(q, hk, hv, np.array(lens), None, scale)
    assert np.isfinite(want).all() and np.isfinite(got).all()
    got, want = (x.reshape(b, seq, group, dk) for x in (got, want))
    # scores, exponentials and sums in float32, as for values of any other size
    dots = max((np.abs(q[i, j].astype(np.float64)) @ np.abs(hk[i, 0]).T).max()
               for i in range(b) for j in range(group)) / scale
    rel = 2 * ((dk + 4) * dots + p + 16) * 2.0**-24 + 2.0**-23
    for i in range(b):
        for blk in range(0, dk, 32):
            s = slice(blk, blk + 32)
            assert np.abs(got[i, ..., s] - want[i, ..., s]).max() <= rel * np.abs(hv[i, ..., s]).max(), (i, blk)
