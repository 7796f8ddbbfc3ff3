"""A table on the host is checked as one on the device."""
import numpy as np
import pytest

from nimbleml_amd import kernels as K
from test_gpu_paged import Cache, queries, upload

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seq", [1, 150])
def test_pages_of_a_row_without_new_tokens_do_not_matter(gpu, seq):
    cache = Cache(3, 1, 32, 8, 30, np.float16, 4)
    q, lens = queries(3, 2, seq, 32, np.float16, 4), np.array([200, 240, 170], np.int32)
    counts = np.array([seq, 0, seq], np.int32)
    want = K.paged_attention(q, cache.c, cache.table, lens, 4.0, counts).numpy()
    bad = cache.table.copy()
    bad[1] = cache.c.num_pages
    for table in (bad, upload(bad)):
        for n in (counts, upload(counts)):
            for at in (lens, upload(lens)):
                assert np.array_equal(K.paged_attention(q, cache.c, table, at, 4.0, n).numpy(), want)
    bad[2, 3] = -1
    for table in (bad, upload(bad)):
        for n in (counts, upload(counts)):
            with pytest.raises(ValueError, match="page"):
                K.paged_attention(q, cache.c, table, lens, 4.0, n)
    none = np.zeros((3, 2, 0, 32), np.float16)
    for table in (bad, upload(bad)):
        assert K.paged_attention(none, cache.c, table, lens, 4.0).shape == (3, 0, 64)
