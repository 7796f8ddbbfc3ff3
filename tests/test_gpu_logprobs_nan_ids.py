"""Alternatives of rows whose first logits are NaN: ids are the row's, NaN first and by id."""
import numpy as np
import pytest

from nimbleml_amd import kernels as K
from oracle import kv4_ref as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("vocab, top_k", [(1, 1), (5, 5), (5, 3), (64, 64), (700, 20), (40000, 7)])
def test_nan_at_the_first_ids(gpu, dtype, vocab, top_k):
    r = np.random.RandomState(vocab)
    x = r.randn(5, vocab).astype(dtype)
    x[0, 0] = np.nan
    x[1] = np.nan
    x[2, [0, vocab - 1]] = np.nan
    x[3, 0], x[3, vocab // 2] = np.nan, np.inf
    x[4, :] = -np.inf
    x[4, 0] = np.nan
    x.view(np.uint16 if dtype == np.float16 else np.uint32)[2, 0] |= 1 << (8 * x.itemsize - 1)  # (−NaN)
    t = np.zeros(5, np.int64)
    logp, _, _, _, ids, top = (a.numpy() for a in K.token_logprobs(x, t, top_k))
    assert np.array_equal(ids, R.logprobs(x, t, top_k)[4])
    assert np.isnan(logp).all() and np.isnan(top).all()
