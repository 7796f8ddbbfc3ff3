"""Attention over pages of scores that are large and differ little: the parts of long rows meet exactly."""
import numpy as np
import pytest

from oracle import draft_ref as R
from test_gpu_paged import Cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("seq, keys, dk", [(1, 5000, 64), (1, 5000, 128), (3, 3000, 32), (150, 3000, 64), (300, 2500, 128),
                                           (260, 2000, 192), (270, 1500, 256), (140, 3000, 96)])
@pytest.mark.parametrize("offset", [0, 32, 256])
def test_scores_near_a_large_one(gpu, seq, keys, dk, dtype, offset):
    """Scores of offset² + x, exact in float32 in any order of the sum, values of one sign for each 200 keys."""
    cache, r = Cache(1, 1, dk, 64, 80, dtype, seq), np.random.RandomState(dk + seq)
    cache.k[:] = r.randint(-2, 3, cache.k.shape) / 4
    q = (r.randint(-2, 3, (1, 2, seq, dk)) / 4).astype(dtype)
    cache.k[..., 0], q[..., 0] = offset, offset
    v = np.where(np.arange(keys) // 200 % 2, 1.0, -1.0)[:, None] * 2.0 ** -r.randint(0, 3, (keys, dk))
    for p in range(keys):
        cache.v[cache.table[0, p // 64], 0, p % 64] = v[p]
    cache.push()
    got = cache.attend(q, np.array([keys], np.int32), scale=1.0).reshape(1, seq, 2, dk).astype(np.float64)
    want, size, _ = R.paged_attention(q, cache.k, cache.v, cache.table, [keys], [seq], 1.0)
    # differences of scores, at most the sum of the other products: their factor to powers of two rounded, the
    # product too, and the sum with the reference; an exponential 2^-23, of each part's merge one more; of a
    # float16 probability 2^-20; all in the products and in the sum of them. A float32 sum rounds once a key at
    # most, and some times in the merge.
    apart = 2 * (dk - 1) / 4 * 1.4427
    lost = size * (2 * 2.0 ** -24 * (3 * apart + 2 + 2) + (2.0 ** -19 if dtype == np.float16 else 0) + 2.0 ** -24 * (keys + 48))
    tol = lost + (2.0 ** -11 if dtype == np.float16 else 2.0 ** -24) * (np.abs(want) + lost) + \
        (2.0 ** -25 if dtype == np.float16 else 0)
    assert (np.abs(got - want) <= tol).all(), (np.abs(got - want) / tol).max()
