"""A workspace that the caller of paged_attention keeps."""
import numpy as np
import pytest

from nimbleml_amd import kernels as K
from test_gpu_paged import Cache, queries

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_one_workspace_for_prompts_and_steps(gpu, dtype):
    cache, r = Cache(4, 2, 64, 16, 140, dtype, 3), np.random.RandomState(3)
    ws = K.paged_attention_workspace(cache.c, 4, 4, 150, 140)
    small = K.paged_attention_workspace(cache.c, 4, 4, 1, 140)
    assert ws.nbytes > small.nbytes > 0
    for i, seq in enumerate((150, 1, 5, 150, 1, 40)):
        q = queries(4, 4, seq, 64, dtype, i)
        lens = r.randint(0, 2241, 4).astype(np.int32)
        lens[i % 4] = 2240
        counts = r.randint(0, seq + 1, 4).astype(np.int32)
        want = K.paged_attention(q, cache.c, cache.table, lens, 8.0, counts).numpy()
        got = K.paged_attention(q, cache.c, cache.table, lens, 8.0, counts, workspace=ws).numpy()
        assert np.array_equal(got, want)
    with pytest.raises(ValueError, match="workspace of"):
        K.paged_attention(queries(4, 4, 150, 64, dtype, 0), cache.c, cache.table, lens, 8.0, workspace=small)
    # none is needed of few keys
    few = Cache(1, 1, 64, 16, 1, dtype, 3)
    none = K.paged_attention_workspace(few.c, 1, 1, 1, 1)
    assert none.nbytes == 0
    K.paged_attention(queries(1, 1, 1, 64, dtype, 0), few.c, few.table, np.array([16], np.int32), 8.0, workspace=none)
