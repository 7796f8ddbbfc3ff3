"""How many keys a call of the paged attention may be over (no GPU needed: the checks come first)."""
import ctypes as C

import pytest

from nimbleml_amd import _native as N

F32, F16 = 0, 1


def workspace(batch, dk, dtype, positions, seq=1):
    need = C.c_size_t()
    N.check(N.lib.nml_paged_attention_workspace(batch, 1, 1, seq, positions // 1024, 1024, dk, dtype, C.byref(need)))
    return need.value


# keys of a span: 16 (float32) or 32 (float16) a wave, two waves a workgroup at head dims 33 … 64, else four; counted
# as 64 at most
@pytest.mark.parametrize("dtype, dk, span", [
    (F32, 32, 64), (F32, 33, 32), (F32, 64, 32), (F32, 65, 64), (F32, 256, 64), (F16, 16, 64), (F16, 64, 64), (F16, 128, 64)])
@pytest.mark.parametrize("positions", [1 << 29, 1 << 30])
def test_the_spans_of_all_rows_are_numbered_in_32_bits(dtype, dk, span, positions):
    most = (2 ** 31 - 1) // (positions // span)  # rows of that many positions
    assert workspace(most, dk, dtype, positions) > 0
    for batch, seq in ((most + 1, 1), (2 * most, 1), (most // 2 + 1, 17)):  # (17 tokens: two tiles of queries)
        with pytest.raises(RuntimeError, match="too many"):
            workspace(batch, dk, dtype, positions, seq)
