"""Verification of drafted tokens reads the rows that a sequence's count gives it, and no others."""
import numpy as np
import pytest

from nimbleml_amd import _native as N
from oracle import draft_ref as R
from test_gpu_verify_drafts import case

pytestmark = pytest.mark.gpu


def call(logits, draft, drafts, u, counts, t, vocab, code):
    """The C call on device arrays of any length: (accepted, tokens, error bits)."""
    batch, n = drafts.shape
    need = N.sz()
    N.check(N.lib.nml_verify_drafts_workspace(batch, n, vocab, N.C.byref(need)))
    d = [None if x is None else N.DeviceArray.from_host(x) for x in (logits, draft, drafts, counts, u)]
    ws = N.DeviceArray.from_host(np.full(need.value, 0xa5, np.uint8))
    a, tok = N.DeviceArray((batch,), np.int32), N.DeviceArray((batch, n + 1), np.int64)
    err = N.DeviceArray.from_host(np.zeros(1, np.int32))
    N.check(N.lib.nml_verify_drafts_device(
        d[0].ptr, vocab, N.ptr(d[1]), vocab, d[2].ptr, N.ptr(d[3]), N.ptr(d[4]), batch, n, vocab, t, a.ptr, tok.ptr,
        ws.ptr, need.value, err.ptr, code))
    return a.numpy(), tok.numpy(), int(err.numpy()[0])


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("t", [1.0, 0.0])
@pytest.mark.parametrize("outright", [False, True])
def test_what_lies_past_a_count(gpu, dtype, t, outright):
    """NaN in the rows of drafts past a count, drafts there that no vocabulary has, numbers that are none."""
    logits, draft, drafts, u, _ = case(6, 5, 3001, dtype, t, seed=21, near=0.2)
    counts = np.array([0, 1, 2, 3, 4, 5], np.int32)
    wa, wt = R.verify(logits, drafts, u, None if outright else draft, counts, t)
    for b, c in enumerate(counts):
        logits[b, c + 1:] = np.nan
        draft[b, c:] = np.nan
        drafts[b, c:] = (-7, 3001, 1 << 40, -1, 1 << 62)[:5 - c]
        u[b, c:5] = np.nan
    a, tok, err = call(logits, None if outright else draft, drafts, u, counts, t, 3001, N.np_dtype_code(dtype))
    assert err == 0 and np.array_equal(a, wa) and np.array_equal(tok, wt)


@pytest.mark.parametrize("t", [0.7, 0.0])
def test_rows_past_the_last_count_need_not_be_there(gpu, t):
    """Buffers that end with the last row that the last sequence's count gives it: the rows that are not there are
    60 of 131072 logits."""
    vocab, n = 1 << 17, 60
    r = np.random.RandomState(22)
    rows = r.randn(n + 2, vocab).astype(np.float32)   # a sequence of n + 1 rows, and the next one's first
    draft = rows[:n] + r.randn(n, vocab).astype(np.float32) * 0.05
    drafts = np.zeros((2, n), np.int64)
    drafts[0], drafts[1] = draft.argmax(-1), vocab - 1
    u, counts = r.rand(2, n + 1), np.array([n, 0], np.int32)
    a, tok, err = call(rows, draft, drafts, u, counts, t, vocab, 0)
    full = np.concatenate([rows, np.zeros((n, vocab), np.float32)]).reshape(2, n + 1, vocab)
    wa, wt = R.verify(full, drafts, u, np.concatenate([draft, draft]).reshape(2, n, vocab), counts, t)
    assert err == 0 and np.array_equal(a, wa) and np.array_equal(tok, wt)


@pytest.mark.parametrize("t", [1.0, 0.0])
@pytest.mark.parametrize("wrong", [-1, 400, -(1 << 40), 1 << 40])
def test_a_draft_out_of_range_behind_a_refusal_is_told(gpu, t, wrong):
    """The first draft is refused, a later one is no token; past a count it does not matter."""
    logits, _, drafts, u, _ = case(3, 4, 400, np.float32, t, seed=23)
    drafts[:, 0] = logits[:, 0].argmin(-1)
    u[:, 0] = 1.0  # (chosen outright: refused unless p = 1)
    counts = np.array([4, 3, 4], np.int32)
    wa, wt = R.verify(logits, drafts, u, None, counts, t)
    assert (wa == 0).all()
    drafts[1, 3] = wrong
    assert call(logits, None, drafts, u, counts, t, 400, 0)[2] == 0
    drafts[2, 3] = wrong
    a, tok, err = call(logits, None, drafts, u, counts, t, 400, 0)
    assert err == 1 and np.array_equal(a, wa) and np.array_equal(tok, wt)
