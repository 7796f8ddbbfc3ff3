"""Verification of drafted tokens on the GPU: whole numbers, equal to the 64-bit statement's."""
import numpy as np
import pytest

from nimbleml_amd import _native as N
from nimbleml_amd import kernels as K
from oracle import draft_ref as R

pytestmark = pytest.mark.gpu


def case(batch, n, vocab, dtype, t=1.0, seed=0, near=0.7):
    """Logits, and drafts drawn from distributions near the target's."""
    r = np.random.RandomState(seed)
    logits = (r.randn(batch, n + 1, vocab) * 2.5).astype(dtype)
    draft = (logits[:, :n] + r.randn(batch, n, vocab) * near).astype(dtype)
    if t > 0:
        q = np.exp(R.log_softmax(draft.reshape(-1, vocab), t)).reshape(batch, n, vocab)
        drafts = (np.cumsum(q, -1) < r.rand(batch, n, 1)).sum(-1).clip(0, vocab - 1)
    else:
        drafts = draft.argmax(-1)
    return logits, draft, drafts.astype(np.int64), r.rand(batch, n + 1), r.randint(0, n + 1, batch)


def check(logits, drafts, u, draft, counts, t):
    a, tok = K.verify_drafts(logits, drafts, u, draft_logits=draft, counts=counts, temperature=t)
    full = np.full(logits.shape[0], logits.shape[1] - 1) if counts is None else counts
    wa, wt = R.verify(logits, drafts, u, draft, full, t)
    assert np.array_equal(a.numpy(), wa) and np.array_equal(tok.numpy(), wt)
    return wa


SIZES = [(1, 1, 1), (1, 4, 7), (3, 5, 1000), (2, 3, 8192), (2, 3, 8193), (33, 2, 257), (1, 63, 40), (2, 1, 130001),
         (4, 8, 32000), (1, 2, 50257)]


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("batch, n, vocab", SIZES)
@pytest.mark.parametrize("t", [1.0, 0.6, 0.0])
def test_verify(gpu, batch, n, vocab, dtype, t):
    logits, draft, drafts, u, counts = case(batch, n, vocab, dtype, t, seed=batch + n + vocab)
    check(logits, drafts, u, draft, None, t)
    check(logits, drafts, u, draft, counts, t)
    check(logits, drafts, u, None, None, t)      # drafts chosen outright
    check(logits, drafts, u, None, counts, t)


def test_no_drafts_is_sampling(gpu):
    logits, _, _, u, _ = case(5, 0, 3000, np.float32)
    a, tok = K.verify_drafts(logits, np.zeros((5, 0), np.int64), u)
    assert (a.numpy() == 0).all()
    p = np.exp(R.log_softmax(logits[:, 0], 1.0))
    assert np.array_equal(tok.numpy()[:, 0], (np.cumsum(p, -1) / p.sum(-1, keepdims=True) <= u).sum(-1))


def test_the_same_distribution_accepts_everything(gpu):
    logits, _, _, u, _ = case(4, 5, 500, np.float16, seed=3)
    drafts = np.random.RandomState(0).randint(0, 500, (4, 5))
    a, tok = K.verify_drafts(logits, drafts, u, draft_logits=logits[:, :5].copy())
    assert (a.numpy() == 5).all() and np.array_equal(tok.numpy()[:, :5], drafts)


def test_a_refusal_that_leaves_nothing(gpu):
    """The draft's distribution is the target's, and a number of 1, out of range, refuses it: the token is
    then one of p's."""
    r = np.random.RandomState(11)
    for vocab in (3, 5000, 20001):
        logits = r.randn(64, 2, vocab).astype(np.float32)
        logits[:, :, 1::2] = -np.inf
        drafts = 2 * r.randint(0, vocab // 2, (64, 1))
        for last in (0.0, 0.3, np.nextafter(1.0, 0.0)):
            u = np.tile([1.0, last], (64, 1))
            a, tok = (x.numpy() for x in K.verify_drafts(logits, drafts, u, draft_logits=logits[:, :1].copy()))
            assert (a == 0).all()
            end = tok[np.arange(64), a]
            assert (end >= 0).all() and (end < vocab).all() and (end % 2 == 0).all()
            p = np.exp(R.log_softmax(logits[np.arange(64), a], 1.0))
            run = np.cumsum(p, -1)[np.arange(64), end]
            assert (run >= last - 1e-9).all() and (run - p[np.arange(64), end] <= last + 1e-9).all()


def test_uniforms_at_the_ends(gpu):
    logits, draft, drafts, u, _ = case(6, 3, 700, np.float32, seed=4)
    for x in (0.0, np.nextafter(1.0, 0.0)):
        check(logits, drafts, np.full_like(u, x), draft, None, 1.0)


def test_ties_and_masked_vocabularies(gpu):
    r = np.random.RandomState(6)
    logits = r.randint(0, 3, (8, 3, 900)).astype(np.float16)  # many equal logits
    drafts = logits[:, :2].argmax(-1).astype(np.int64)
    drafts[4:, 1] += 1
    u = r.rand(8, 3)
    check(logits, drafts, u, None, None, 0.0)
    logits[:, :, 300:] = -np.inf
    logits[0, :, :299] = -np.inf  # one token left
    drafts[0] = 299
    draft = logits[:, :2].copy()
    draft[1, 0, :100] = -np.inf   # a token that the draft never gives
    check(logits, drafts, u, draft, None, 1.0)
    check(logits, drafts, u, None, None, 1.0)
    check(logits, drafts, u, None, None, 0.0)
    logits[:] = np.finfo(np.float16).min
    check(logits, drafts, u, None, None, 1.0)
    check(logits, drafts, u, None, None, 0.0)


def test_large_logits(gpu):
    """Differences of float32 logits near its largest."""
    r = np.random.RandomState(7)
    # (4.5 standard deviations, more than 2400 numbers reach, are 3.4e38, which float32 holds)
    logits = (r.randn(3, 2, 400) * 7.5e37).astype(np.float32)
    drafts = logits[:, :1].argmax(-1).astype(np.int64)
    check(logits, drafts, r.rand(3, 2), None, None, 1.0)
    check(logits * 1e-3, drafts, r.rand(3, 2), (logits[:, :1] * 1e-3), None, 1e6)


def test_tokens_are_distributed_as_the_target(gpu):
    r = np.random.RandomState(8)
    p_logits, q_logits = r.randn(2, 12).astype(np.float32), r.randn(12).astype(np.float32)
    batch = 20000
    q = np.exp(R.log_softmax(q_logits[None], 1.0))[0]
    drafts = r.choice(12, (batch, 1), p=q / q.sum())
    u = r.rand(batch, 2)
    a, tok = K.verify_drafts(np.tile(p_logits, (batch, 1, 1)), drafts, u,
                             draft_logits=np.tile(q_logits, (batch, 1, 1)))
    p = np.exp(R.log_softmax(p_logits, 1.0))
    first = np.bincount(tok.numpy()[:, 0], minlength=12) / batch
    assert (np.abs(first - p[0]) < 5 * np.sqrt(p[0] * (1 - p[0]) / batch)).all()
    two = tok.numpy()[a.numpy() == 1, 1]
    assert (np.abs(np.bincount(two, minlength=12) / len(two) - p[1]) <
            5 * np.sqrt(p[1] * (1 - p[1]) / len(two))).all()


def raw(logits, drafts, u, draft, counts, t, ld=None):
    """The C call: (accepted, tokens, error bits)."""
    batch, n1, vocab = logits.shape
    need = N.sz()
    N.check(N.lib.nml_verify_drafts_workspace(batch, n1 - 1, vocab, N.C.byref(need)))
    d = [N.DeviceArray.from_host(x) if x is not None else None for x in
         (logits, draft, np.asarray(drafts, np.int64), counts, u)]
    ws = N.DeviceArray.from_host(np.full(need.value, 0xa5, np.uint8))  # (in any state)
    a, tok = N.DeviceArray((batch,), np.int32), N.DeviceArray((batch, n1), np.int64)
    err = N.DeviceArray.from_host(np.zeros(1, np.int32))
    N.check(N.lib.nml_verify_drafts_device(
        d[0].ptr, vocab, N.ptr(d[1]), vocab, d[2].ptr, N.ptr(d[3]), N.ptr(d[4]), batch, n1 - 1, vocab, t,
        a.ptr, tok.ptr, ws.ptr, need.value, err.ptr, N.np_dtype_code(logits.dtype)))
    return a.numpy(), tok.numpy(), int(err.numpy()[0])


@pytest.mark.parametrize("t", [1.0, 0.0])
def test_rows_without_a_distribution(gpu, t):
    r = np.random.RandomState(9)
    logits = r.randn(5, 3, 300).astype(np.float32)
    drafts = logits[:, :2].argmax(-1)
    draft = (logits[:, :2] + 1).copy()  # (the same distribution: everything is accepted)
    u = r.rand(5, 3)
    logits[0, 1, 7] = np.nan
    logits[1, 2] = -np.inf
    if t > 0:
        logits[2, 0, 5] = np.inf
        draft[3, 1, 5] = np.nan
    a, tok, err = raw(logits, drafts, u, draft, None, t)
    assert err == 2
    assert a[0] == 1 and tok[0].tolist() == [drafts[0, 0], -1, -1]
    assert a[1] == 2 and tok[1].tolist() == [*drafts[1], -1]
    if t > 0:
        assert a[2] == 0 and (tok[2] == -1).all()
        assert a[3] == 1 and tok[3].tolist() == [drafts[3, 0], -1, -1]
    assert a[4] == 2 and tok[4, 2] >= 0
    with pytest.raises(ValueError, match="NaN"):
        K.verify_drafts(logits, drafts, u, draft_logits=draft, temperature=t)


@pytest.mark.parametrize("t", [1.0, 0.0])
def test_counts_and_drafts_out_of_range(gpu, t):
    logits, draft, drafts, u, _ = case(4, 3, 200, np.float32, t, seed=10, near=0.0)
    drafts[1, 1] = 200
    drafts[2, 0] = -1
    counts = np.array([9, 3, 3, -4], np.int32)
    a, tok, err = raw(logits, drafts, u, draft, counts, t)
    assert err == 1
    fixed = np.array([3, 1, 0, 0])
    wa, wt = R.verify(logits, np.clip(drafts, 0, 199), u, draft, fixed, t)
    assert a[0] == wa[0] and np.array_equal(tok[0], wt[0])
    assert a[1] == 1 and a[2] == 0 and a[3] == 0 and (tok[3, 1:] == -1).all()
    assert (tok[[1, 2], [1, 0]] >= 0).all() and (tok[[1, 2], [1, 0]] < 200).all()
    with pytest.raises(ValueError, match="outside"):
        K.verify_drafts(logits, drafts, u, draft_logits=draft, temperature=t)
