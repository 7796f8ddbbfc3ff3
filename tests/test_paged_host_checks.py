"""What the paged attention's wrapper refuses by itself (no GPU needed: the checks come first)."""
import numpy as np
import pytest

from nimbleml_amd import kernels as K


class Pages:
    """A cache's sizes alone."""
    num_pages, page_size, kv_heads, dk, dtype = 4, 16, 1, 32, np.dtype(np.float32)


def test_pages_of_rows_that_do_not_attend_are_not_looked_at():
    table = np.array([[3, 1], [9, -1]])
    K._check_pages("x", table, [32, 16], 16, 4, [1, 0])
    with pytest.raises(ValueError, match="page 9"):
        K._check_pages("x", table, [32, 16], 16, 4, [0, 1])
    with pytest.raises(ValueError, match="needs 3 pages"):  # (a length is wrong of any row)
        K._check_pages("x", table, [32, 48], 16, 4, [1, 0])


@pytest.mark.parametrize("lens, counts, match", [
    (5, None, "lens must be"), ([5], None, "lens must be"), ([5, 5, 5], None, "lens must be"),
    ([5, 5], [1], "counts must be"), ([5, 5], 1, "counts must be")])
def test_shapes(lens, counts, match):
    q, table = np.zeros((2, 1, 1, 32), np.float32), np.zeros((2, 2), np.int32)
    with pytest.raises(ValueError, match=match):
        K.paged_attention(q, Pages, table, lens, 4.0, counts)
