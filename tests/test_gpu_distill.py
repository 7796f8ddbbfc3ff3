"""Distillation from a teacher's top logits on the GPU against its 64-bit statement."""
import numpy as np
import pytest

import nimbleml_amd as nm
from nimbleml_amd import _native as N
from nimbleml_amd import kernels as K
from oracle import draft_ref as R

pytestmark = pytest.mark.gpu

EPS = {np.float32: 2.0 ** -24, np.float16: 2.0 ** -11}  # half a step, relative


def case(rows, vocab, k, dtype, seed=0, absent=True, std=2.5):
    r = np.random.RandomState(seed)
    x = (r.randn(rows, vocab) * std).astype(dtype)
    ids = np.stack([r.choice(vocab, k, replace=k > vocab) for _ in range(rows)]).astype(np.int64)
    y = (np.take_along_axis(x.astype(np.float32), ids, -1) + r.randn(rows, k) * 0.7).astype(np.float32)
    if absent:
        ids[::5] = -1                 # no teacher
        ids[1::5, k // 2:] = -1
        y[2::5, 0] = -np.inf          # absent as well
        if k > 2:
            ids[3::5, 2] = ids[3::5, 0]  # the same id twice
    return x, ids, y, r.randn(rows).astype(np.float32)


def tolerances(x, t):
    """An exponent (x − m)/T is rounded three times (the difference, the factor log₂ e / T, the product) to
    2^-24 of itself, S at most: its exponential is off by 3·S·2^-24 and a last place. A loss is a sum of
    terms of at most S (or the teacher's as much, which adds 2 here) and of two logarithms of sums."""
    s = (x.astype(np.float64).max(-1) - x.astype(np.float64).min(-1)) / t + 4
    return 2.0 ** -24 * (3 * s + 8), 2.0 ** -24 * (16 * s + 32)


SIZES = [(1, 1, 1), (1, 7, 3), (3, 100, 5), (2, 50257, 20), (5, 4096, 64), (7, 1001, 256), (600, 333, 20),
         (1, 130001, 100), (4, 8193, 1), (9, 255, 7)]


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("rows, vocab, k", SIZES)
@pytest.mark.parametrize("t", [1.0, 2.3])
def test_distill_and_gradient(gpu, rows, vocab, k, dtype, t):
    x, ids, y, dloss = case(rows, vocab, k, dtype, seed=rows + vocab, absent=rows > 1)
    loss, m, l = (a.numpy() for a in K.distill(x, ids, y, t))
    want, wm, wl = R.distill(x, ids, y, t)
    tol_l, tol = tolerances(x, t)
    assert np.array_equal(m, wm.astype(np.float32))
    assert (np.abs(l - wl) <= tol_l * wl).all()
    assert (np.abs(loss - want) <= tol).all()
    got = K.distill_backward(x, ids, y, m, l, dloss, t).numpy().astype(np.float64)
    grad, p, q = R.distill_grad(x, ids, y, dloss, t)
    scale = np.abs(dloss.astype(np.float64) / t)[:, None]
    # p and q are off by their exponents' roundings and their sums'; the result is rounded once
    # (float16 below 2^-14: to half of 2^-24)
    tol = scale * (p + q) * 2 * tol_l[:, None] + EPS[dtype] * np.abs(grad) + (2.0 ** -25 if dtype == np.float16 else 1e-44)
    assert (np.abs(got - grad) <= tol).all()
    none = ~((ids >= 0) & (y > -np.inf)).any(-1)
    assert (loss[none] == 0).all() and (got[none] == 0).all()


def test_rows_at_a_stride_and_in_place(gpu):
    """Logits at an odd stride, the gradient written over them; what lies between the rows stays."""
    x, ids, y, dloss = case(6, 1003, 9, np.float16, seed=3)
    ld = 1017
    wide = np.full((6, ld), 7.0, np.float16)
    wide[:, :1003] = x
    buf, di, dy, dd = (N.DeviceArray.from_host(a) for a in (wide, ids, y, dloss))
    stats = [N.DeviceArray((6,), np.float32) for _ in range(3)]
    N.check(N.lib.nml_distill_device(buf.ptr, ld, di.ptr, dy.ptr, 6, 1003, 9, 1.5, *(s.ptr for s in stats), None, 1))
    N.check(N.lib.nml_distill_backward_device(buf.ptr, ld, di.ptr, dy.ptr, stats[1].ptr, stats[2].ptr, dd.ptr, 6,
                                              1003, 9, 1.5, buf.ptr, ld, None, 1))
    alone = K.distill_backward(x, ids, y, stats[1], stats[2], dloss, 1.5).numpy()
    got = buf.numpy()
    assert np.array_equal(got[:, :1003], alone)
    assert (got[:, 1003:] == 7.0).all()


def test_infinities_and_nan(gpu):
    r = np.random.RandomState(5)
    x = r.randn(8, 300).astype(np.float32)
    ids = np.tile(np.arange(4), (8, 1)).astype(np.int64)
    y = r.randn(8, 4).astype(np.float32)
    x[0, 2] = -np.inf          # q > 0 where p = 0
    x[1, 100] = np.nan
    x[2, 100] = np.inf
    x[3] = -np.inf
    y[4, 1] = np.nan
    y[5, 1] = np.inf
    x[6, 50:] = -np.inf        # a masked vocabulary
    x[7] = np.finfo(np.float32).min  # all of the type's lowest value: uniform
    loss, m, l = K.distill(x, ids, y)
    got = loss.numpy()
    assert got[0] == np.inf and np.isnan(got[1:6]).all()
    want = R.distill(x[6:], ids[6:], y[6:], 1.0)[0]
    assert np.allclose(got[6:], want, rtol=0, atol=1e-5)
    d = K.distill_backward(x, ids, y, m, l, np.ones(8, np.float32)).numpy()
    assert np.isnan(d[1]).all() and np.isnan(d[3]).all() and np.isnan(d[4]).all() and np.isnan(d[5]).all()
    assert np.isfinite(d[[0, 6, 7]]).all() and (d[6, 50:] == 0).all()


def test_ids_out_of_range_are_told(gpu):
    x, ids, y, dloss = case(4, 60, 3, np.float32, absent=False)
    for bad in (60, -2, 1 << 40):
        ids[2, 1] = bad
        with pytest.raises(ValueError, match="outside"):
            K.distill(x, ids, y)
        with pytest.raises(ValueError, match="outside"):
            K.distill_backward(x, ids, y, np.zeros(4, np.float32), np.ones(4, np.float32), dloss)


def test_offsets_cost_nothing(gpu):
    """The teacher's logits and log probabilities, and large ones, give the same loss."""
    x, ids, y, _ = case(20, 500, 8, np.float32, seed=8, absent=False)
    ref = K.distill(x, ids, y)[0].numpy()
    for shift in (np.float32(64.0), np.float32(-1024.0)):
        got = K.distill(x, ids, y + shift)[0].numpy()
        # (y itself is rounded by the addition, 2^-24·1024 at most)
        assert np.abs(got - ref).max() <= 2.0 ** -24 * 1024 * 4


def test_one_teacher_token_is_its_log_probability(gpu):
    x, _, _, dloss = case(50, 777, 1, np.float32, seed=9)
    ids = np.random.RandomState(1).randint(0, 777, (50, 1))
    loss, m, l = K.distill(x, ids, np.full((50, 1), 3.0, np.float32))
    lp = K.token_logprobs(x, ids[:, 0])
    tol = tolerances(x, 1.0)[1]
    assert (np.abs(loss.numpy() + lp[0].numpy()) <= 2 * tol).all()
    a = K.distill_backward(x, ids, np.zeros((50, 1), np.float32), m, l, dloss).numpy()
    b = K.token_logprobs_backward(x, ids[:, 0], lp[2], lp[3], None, -dloss).numpy()
    assert (np.abs(a - b) <= np.abs(dloss)[:, None] * 2 * tol[:, None]).all()


def test_loss_tensor_and_its_backward(gpu):
    """distill_loss of a model's logits: its gradient at the logits is the formula's, and goes on into
    the parameters as the logits' own backward takes it there."""
    nm.set_dtype("float32")
    np.random.seed(0)
    teacher, student = nm.GPT(96, 32, 4, 2, 24), nm.GPT(96, 16, 2, 1, 24)
    ids = np.random.randint(0, 96, (2, 24))
    top = teacher.log_probs(ids, np.zeros((2, 24), np.int64), top_k=10)
    logits = student.forward(ids)
    loss = nm.distill_loss(logits, top["top_ids"], top["top_logp"], temperature=2.0)
    x = np.asarray(logits.data).reshape(48, 96)
    ti, tl = top["top_ids"].numpy().reshape(48, 10), top["top_logp"].numpy().reshape(48, 10)
    assert np.allclose(np.asarray(loss.data).reshape(-1), R.distill(x, ti, tl, 2.0)[0], atol=1e-5)
    w = np.random.rand(2, 24).astype(np.float32)
    loss.backward(w)
    d = R.distill_grad(x, ti, tl, w.reshape(-1), 2.0)[0].astype(np.float32)
    assert np.allclose(np.asarray(logits.grad).reshape(48, 96), d, atol=1e-6)
    got = {n: p.grad.copy() for n, p in nm.named_parameters(student)}
    for _, p in nm.named_parameters(student):
        p.zero_grad(set_to_none=True)
    again = student.forward(ids)
    again.backward(d.reshape(2, 24, 96))
    for n, p in nm.named_parameters(student):
        assert np.allclose(got[n], p.grad, atol=1e-5 * max(1.0, np.abs(p.grad).max())), n


def test_loss_without_gradients(gpu):
    nm.set_dtype("float32")
    x = nm.Tensor(np.zeros((3, 8), np.float32), (3, 8))
    with nm.no_grad():
        out = nm.distill_loss(x, np.zeros((3, 2), np.int64), np.zeros((3, 2), np.float32))
    # (two entries of one id, each of q = 1/2: log 1/2 − log 1/8)
    assert not out.requires_grad and np.allclose(np.asarray(out.data), np.log(4.0), atol=1e-6)
