"""Distillation of logits that lie further apart than float32's largest value."""
import numpy as np
import pytest

from nimbleml_amd import kernels as K
from oracle import draft_ref as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab, top_k", [(7, 3), (5000, 256)])
@pytest.mark.parametrize("t", [4.0, 1e3, 1e6])
def test_logits_far_apart(gpu, t, vocab, top_k):
    """Masks of the type's lowest value beside large logits: the differences reach twice float32's largest, the
    divergence does not."""
    r = np.random.RandomState(vocab)
    rows = 6
    x = r.uniform(-3.0e38, 3.0e38, (rows, vocab)).astype(np.float32)
    x[:, ::3] = np.finfo(np.float32).min
    x[:, 1] = 3.3e38
    ids = np.stack([r.permutation(vocab)[:top_k] for _ in range(rows)]).astype(np.int64)
    ids[0], ids[1, 0] = 0, 1  # (one row of nothing but a masked token)
    y = r.randn(rows, top_k).astype(np.float32)
    loss = K.distill(x, ids, y, t)[0].numpy().astype(np.float64)
    want = R.distill(x, ids, y, t)[0]
    assert np.isfinite(want).all() and want.max() < 3.4e38
    # all terms are of one sign (log p ≤ 0, and what log q adds is nothing beside it): a rounding of the logits'
    # difference, of the product with q, of q (an exponential, 2^-23, and its argument, 2^-24 of 8 at most), of 1/T,
    # of the quotient and the product, and one for each of the sums' 9 steps, twice
    assert (np.abs(loss - want) <= np.abs(want) * 2.0 ** -24 * (5 + 2 + 8 + 2 * 9 + 8)).all()
