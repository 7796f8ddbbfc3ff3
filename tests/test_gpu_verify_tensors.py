"""Verification takes what a model's cached forward returns."""
import numpy as np
import pytest

import nimbleml_amd as nm
from nimbleml_amd import kernels as K

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("t", [0.8, 0.0])
def test_logits_of_a_cached_forward(gpu, dtype, t):
    nm.set_dtype(dtype)
    try:
        np.random.seed(1)
        target, drafter = nm.GPT(96, 64, 4, 2, 32), nm.GPT(96, 32, 2, 1, 32)
        r = np.random.RandomState(2)
        ids = r.randint(0, 96, (2, 5))
        logits, _ = target.forward_with_cache(ids, nm.KVCache(target, 2))
        seen, _ = drafter.forward_with_cache(ids[:, :4], nm.KVCache(drafter, 2))
        assert isinstance(logits, nm.Tensor) and logits.shape == (2, 5, 96) and seen.shape == (2, 4, 96)
        u, drafts = r.rand(2, 5), ids[:, 1:]
        got = K.verify_drafts(logits, drafts, u, draft_logits=seen, temperature=t)
        want = K.verify_drafts(logits.data.reshape(2, 5, 96), drafts, u, draft_logits=np.asarray(seen.data).reshape(2, 4, 96),
                               temperature=t)
        for x, y in zip(got, want):
            assert np.array_equal(x.numpy(), y.numpy())
        # and of a Tensor whose values are on the host
        host = nm.Tensor(logits.data.numpy(), logits.shape)
        a, _ = K.verify_drafts(host, drafts, u, draft_logits=nm.Tensor(seen.data.numpy(), seen.shape), temperature=t)
        assert np.array_equal(a.numpy(), got[0].numpy())
    finally:
        nm.set_dtype("float32")
