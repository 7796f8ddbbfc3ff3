"""Token log probabilities, entropies, alternatives and their gradient against 64-bit statements
(oracle/kv4_ref.py) and against differences."""
import numpy as np
import pytest

from nimbleml_amd import _native as N
from nimbleml_amd import kernels as K
from oracle import kv4_ref as R

pytestmark = pytest.mark.gpu

DTYPES = [np.float16, np.float32]


def logits_of(r, rows, vocab, dtype, std=3.0):
    return (std * r.randn(rows, vocab)).astype(dtype)


def tol_of(x):
    """A float32 statistic of logits x: t = x − max is exact to 2^-24 of |x|, its exponential to
    (2 + |t|)·2^-23 relative, weighted by p where |t|·p ≤ 1, sums of V terms in trees of at most
    400 additions deep; log Z and the result round once more."""
    big = np.abs(x[np.isfinite(x)]).max() + np.log(x.shape[1])
    return 2.0**-23 * (2 * big + 2 * np.log(x.shape[1]) + 400 / 8 + 4)


def check(x, t, top_k=0, ignore=None):
    got = [None if a is None else a.numpy() for a in K.token_logprobs(x, t, top_k, ignore)]
    want = R.logprobs(x, t, top_k, ignore)
    assert np.array_equal(got[2], want[2].astype(np.float32), equal_nan=True) or np.isnan(want[3]).any()
    for g, w in zip((got[0], got[1], got[3] / np.maximum(want[3], 1)), (want[0], want[1], want[3] / np.maximum(want[3], 1))):
        assert np.array_equal(np.isnan(g), np.isnan(w))
        inf = np.isinf(w)
        assert np.array_equal(g[inf], w[inf].astype(np.float32))
        ok = np.isfinite(w)
        assert ok.sum() == 0 or np.abs(g[ok] - w[ok]).max() <= tol_of(x)
    if top_k:
        assert np.array_equal(got[4], want[4])
        assert np.array_equal(np.isnan(got[5]), np.isnan(want[5]))
        fin = np.isfinite(want[5])
        assert np.array_equal(got[5][np.isinf(want[5])], want[5][np.isinf(want[5])])
        assert fin.sum() == 0 or np.abs(got[5][fin] - want[5][fin]).max() <= tol_of(x)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 63, 64, 65, 257, 1000, 1023, 4096, 8191, 8200, 16391,
                                   32000, 50257, 65537, 131100])
def test_every_vocabulary_size(gpu, dtype, vocab):
    r = np.random.RandomState(vocab)
    x = logits_of(r, 5, vocab, dtype)
    check(x, r.randint(0, vocab, 5), min(vocab, 20))
    check(x, r.randint(0, vocab, 5), min(vocab, 64))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("top_k", [1, 2, 5, 33, 50])
def test_alternatives_with_equal_logits(gpu, dtype, top_k):
    """Few distinct values: ties go to the lower id; all equal, all masked but a few."""
    r = np.random.RandomState(top_k)
    x = np.round(logits_of(r, 6, 3001, dtype, 1.5)).astype(dtype)
    x[1] = 0.5
    x[2] = -np.inf
    x[2, [5, 77, 2999]] = [1, 3, 3]
    x[3, ::2] = -0.0
    x[3, 1::2] = 0.0
    x[4, :2900] = -np.inf
    check(x, np.array([0, 5, 77, 3, 2950, 3000]), top_k)


@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_infinite_and_nan_logits(gpu, dtype):
    r = np.random.RandomState(2)
    x = logits_of(r, 8, 500, dtype)
    x[0, 100:] = -np.inf           # masked: probability 0, nothing added
    x[1, 7] = -np.inf              # the target itself is masked: logp −inf
    x[2] = -np.inf                 # nothing left: NaN
    x[3, 9] = np.nan
    x[4, 11] = np.inf
    x[5] = np.finfo(dtype).min     # the type's lowest value everywhere: uniform
    x[6, 1:] = np.finfo(dtype).min
    t = np.array([3, 7, 0, 0, 0, 4, 0, 1])
    got = K.token_logprobs(x, t)
    for a in got[:2]:
        assert np.array_equal(np.isnan(a.numpy()), [False, False, True, True, True, False, False, False])
    assert got[0].numpy()[1] == -np.inf
    assert abs(got[0].numpy()[5] + np.log(500)) <= 1e-6 and got[0].numpy()[6] == 0
    assert got[1].numpy()[6] == 0
    d = K.token_logprobs_backward(x, t, got[2], got[3], got[1], np.ones(8, np.float32)).numpy()
    # the uniform row's gradient: 1 at the target less 1/500 everywhere, a step of the type off
    want = (np.arange(500) == 4) - 1 / 500
    assert np.abs(d[5].astype(np.float64) - want).max() <= np.finfo(dtype).eps / 2 + 1e-6
    keep = [0, 1, 5, 6, 7]
    check(x[keep], t[keep], 20)
    check(x[[2, 3]], t[[2, 3]], 5)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_and_unaligned_rows_keep_what_lies_between(gpu, dtype):
    """Rows of 1001 logits at a stride of 1013, the first of them off any 16-byte line."""
    r = np.random.RandomState(3)
    v, ld, rows, off = 1001, 1013, 7, 3
    flat = logits_of(r, 1, off + ld * rows, dtype)[0]
    flat[off + v::ld] = np.nan
    dev = N.DeviceArray.from_host(flat)
    x = np.stack([flat[off + i * ld: off + i * ld + v] for i in range(rows)])
    t = r.randint(0, v, rows)
    td = N.DeviceArray.from_host(t.astype(np.int64))
    lp, en, m, ls = (N.DeviceArray((rows,), np.float32) for _ in range(4))
    p, code = dev.ptr + off * flat.itemsize, N.np_dtype_code(dtype)
    N.check(N.lib.nml_token_logprobs_device(p, ld, td.ptr, rows, v, 0, 0, 0, lp.ptr, en.ptr, m.ptr,
                                            ls.ptr, None, None, None, code))
    want = R.logprobs(x, t)
    for g, w in zip((lp, en, m), want):
        assert np.abs(g.numpy() - w).max() <= tol_of(x)
    assert np.abs(ls.numpy() / want[3] - 1).max() <= tol_of(x)
    # the gradient into rows of another stride and alignment, then over the logits themselves
    dl = r.randn(rows).astype(np.float32)
    dld = N.DeviceArray.from_host(dl)
    ld2 = 1006
    out = N.DeviceArray.from_host(np.full(1 + ld2 * rows, 9, dtype))
    N.check(N.lib.nml_token_logprobs_backward_device(
        p, ld, td.ptr, m.ptr, ls.ptr, en.ptr, dld.ptr, None, rows, v, 0, 0, out.ptr + flat.itemsize, ld2, None,
        code))
    got = out.numpy()[1:].reshape(rows, ld2)
    assert (got[:, v:] == 9).all() and out.numpy()[0] == 9
    N.check(N.lib.nml_token_logprobs_backward_device(
        p, ld, td.ptr, m.ptr, ls.ptr, en.ptr, dld.ptr, None, rows, v, 0, 0, p, ld, None, code))
    over = dev.numpy()
    for i in range(rows):
        assert np.array_equal(over[off + i * ld: off + i * ld + v], got[i, :v])
        end = slice(off + i * ld + v, off + (i + 1) * ld)
        assert np.array_equal(over[end], flat[end], equal_nan=True)
    assert np.array_equal(over[:off], flat[:off])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, vocab", [(1, 1), (3, 5), (9, 640), (4, 32001), (2, 70000)])
def test_gradient(gpu, dtype, rows, vocab):
    r = np.random.RandomState(rows)
    x = logits_of(r, rows, vocab, dtype)
    x[0, vocab // 2:] = -np.inf if vocab > 2 else x[0, vocab // 2:]
    t = r.randint(0, max(1, vocab // 3), rows)
    dl, dh = r.randn(rows).astype(np.float32), r.randn(rows).astype(np.float32)
    ignore = int(t[-1]) if rows > 2 else None
    lp, en, m, ls, _, _ = K.token_logprobs(x, t, 0, ignore)
    got = K.token_logprobs_backward(x, t, m, ls, en, dl, dh, ignore).numpy().astype(np.float64)
    want = R.logprobs_grad(x, t, dl.astype(np.float64), dh.astype(np.float64), ignore)
    # p to (|log p| + 4)·2^-23 relative from the statistics' error and the exponential's; |log p|·p ≤ 0.4
    big = np.abs(x[np.isfinite(x)]).max() + np.log(vocab)
    scale = np.abs(dl).max() + np.abs(dh).max() * (1 + np.log(vocab))
    tol = scale * (2 * tol_of(x) + 4 * 2.0**-23 * (big + 4)) + np.finfo(dtype).eps / 2 * np.abs(want).max()
    assert np.abs(got - want).max() <= tol + np.finfo(dtype).tiny
    only = K.token_logprobs_backward(x, t, m, ls, en, dl, None, ignore).numpy().astype(np.float64)
    assert np.abs(only - R.logprobs_grad(x, t, dl, np.zeros(rows), ignore)).max() <= tol
    none = K.token_logprobs_backward(x, t, m, ls, en, None, None, ignore).numpy()
    assert (none == 0).all()


def test_gradient_against_differences(gpu):
    r = np.random.RandomState(5)
    x = logits_of(r, 3, 40, np.float32, 1.0)
    t, dl, dh = np.array([1, 20, 39]), r.randn(3), r.randn(3)

    def f(y):
        lp, en, *_ = R.logprobs(y, t)
        return (dl * lp + dh * en).sum()

    lp, en, m, ls, _, _ = K.token_logprobs(x, t)
    got = K.token_logprobs_backward(x, t, m, ls, en, dl.astype(np.float32),
                                    dh.astype(np.float32)).numpy()
    h = 1e-5
    for i in range(3):
        for j in range(0, 40, 3):
            up, down = x.astype(np.float64), x.astype(np.float64)
            up[i, j] += h
            down[i, j] -= h
            d = (f(up) - f(down)) / (2 * h)  # off by h²·|f'''| / 6 < 1e-9 and 1e-16·|f| / h < 1e-9
            assert abs(got[i, j] - d) <= 1e-5


@pytest.mark.parametrize("dtype", DTYPES)
def test_ignored_rows_and_targets_out_of_range(gpu, dtype):
    r = np.random.RandomState(6)
    x = logits_of(r, 6, 300, dtype)
    t = np.array([5, -100, 299, -100, 0, 7])
    x[1] = np.nan  # an ignored row is not read
    check(x[[0, 2, 3, 4, 5]], t[[0, 2, 3, 4, 5]], 4, -100)
    lp, en, m, ls, ids, top = K.token_logprobs(x, t, 4, -100)
    assert lp.numpy()[1] == 0 and en.numpy()[1] == 0 and (ids.numpy()[1] == -1).all()
    d = K.token_logprobs_backward(x, t, m, ls, en, np.ones(6, np.float32), None, -100).numpy()
    assert (d[[1, 3]] == 0).all() and np.isfinite(d).all()
    for bad in (300, -1, 2**40):
        t[4] = bad
        with pytest.raises(ValueError, match="out of range"):
            K.token_logprobs(x, t, 0, -100)
        with pytest.raises(ValueError, match="out of range"):
            K.token_logprobs_backward(x, t, m, ls, en, np.ones(6, np.float32), None, -100)


def test_statistics_alone(gpu):
    """No targets: entropies, log sums and alternatives of the logits themselves."""
    r = np.random.RandomState(7)
    x = logits_of(r, 4, 999, np.float16)
    dev = N.DeviceArray.from_host(x)
    en, ids, top = N.DeviceArray((4,), np.float32), N.DeviceArray((4, 3), np.int64), N.DeviceArray((4, 3), np.float32)
    N.check(N.lib.nml_token_logprobs_device(dev.ptr, 999, None, 4, 999, 0, 1, 3, None, en.ptr, None, None,
                                            ids.ptr, top.ptr, None, N.F16))
    want = R.logprobs(x, np.zeros(4, np.int64), 3)
    assert np.array_equal(ids.numpy(), want[4])
    assert np.abs(en.numpy() - want[1]).max() <= tol_of(x) and np.abs(top.numpy() - want[5]).max() <= tol_of(x)


def test_more_rows_than_one_launch_takes(gpu):
    """2^21 + 5 rows: the first, the last and those at the seam are their own."""
    r = np.random.RandomState(31)
    rows, vocab = (1 << 21) + 5, 5
    x = logits_of(r, rows, vocab, np.float16)
    t = r.randint(0, vocab, rows)
    t[-2] = 1 << 40  # ignored
    got = [a.numpy() for a in K.token_logprobs(x, t, 2, 1 << 40)]
    for s in (slice(0, 9), slice((1 << 21) - 7, rows)):
        # (not bit for bit those of a call of their own: a row's sums are grouped by where its
        # 16-byte pieces begin)
        want = R.logprobs(x[s], t[s], 2, 1 << 40)
        for g, w in zip(got, want):
            assert g[s].shape == w.shape and np.abs(g[s] - w).max() <= tol_of(x[s]) * np.maximum(1, np.abs(w).max())
        assert np.array_equal(got[4][s], want[4])
