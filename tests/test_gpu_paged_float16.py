"""Float16 attention over pages keeps the probabilities' bits, for one new token and for many: outputs that
small differences of probabilities make up are off by no more than float32 sums and their own rounding."""
import numpy as np
import pytest

from oracle import draft_ref as R
from test_gpu_paged import Cache

pytestmark = pytest.mark.gpu


# (kv heads, queries a KV head, head dim, page, pages, new tokens, keys)
@pytest.mark.parametrize("kv, group, dk, page, pages, seq, keys", [
    (2, 4, 128, 64, 5, 1, 310), (2, 4, 128, 64, 5, 8, 310), (2, 4, 128, 64, 5, 9, 310), (1, 4, 128, 64, 8, 300, 301),
    (2, 1, 64, 16, 20, 129, 222), (1, 3, 96, 32, 9, 200, 264), (1, 2, 192, 64, 4, 90, 250), (1, 1, 256, 16, 20, 150, 300),
    (1, 1, 72, 8, 40, 40, 41)])
def test_differences_of_probabilities(gpu, kv, group, dk, page, pages, seq, keys):
    cache, heads, r = Cache(1, kv, dk, page, pages, np.float16), kv * group, np.random.RandomState(dk + seq)
    # quarters, whose products float32 adds exactly; values of either sign in turn, so that outputs are differences
    q = (r.randint(-4, 5, (1, heads, seq, dk)) / 4).astype(np.float16)
    cache.k[:] = r.randint(-4, 5, cache.k.shape) / 4
    for p in range(keys):
        cache.v[cache.table[0, p // page], :, p % page] = (-1) ** p * 2.0 ** -r.randint(0, 3, (kv, dk))
    cache.push()
    got = cache.attend(q, np.array([keys], np.int32)).reshape(1, seq, heads, dk).astype(np.float64)
    want, size, _ = R.paged_attention(q, cache.k, cache.v, cache.table, [keys], [seq], np.sqrt(dk))
    k = np.concatenate([cache.k[i].astype(np.float64) for i in cache.table[0]], 1)[:, :keys]
    score = max(np.abs(q[0, h].astype(np.float64) @ k[h // group].T).max() for h in range(heads)) / np.sqrt(dk)
    # a score is rounded with its factor, the factor itself and its reference: 2^-24 of it four times; an
    # exponential is off by 2^-23; of a probability 2^-20 may be lost; all of it in the products and in Σ p. A
    # float32 sum is rounded once a key at most, and some times in the merge. Then the output's rounding.
    lost = size * (2 * 2.0 ** -24 * (4 * score + 2) + 2.0 ** -19 + 2.0 ** -24 * (keys + 32))
    tol = lost + 2.0 ** -11 * (np.abs(want) + lost) + 2.0 ** -25
    assert (np.abs(got - want) <= tol).all(), (np.abs(got - want) / tol).max()
