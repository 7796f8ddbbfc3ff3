"""``token_log_probs`` in float16 mode: the gradient given to its float32 output reaches the kernel as
it was given."""
import numpy as np
import pytest

import nimbleml_amd as nm
from nimbleml_amd import _native as N
from nimbleml_amd import np_backend
from nimbleml_amd.tensor import Tensor
from oracle import kv4_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture
def half():
    before = np_backend.dtype
    nm.set_dtype("float16")
    yield
    nm.set_dtype(np.dtype(before).name)


def test_upstream_gradients_past_float16(gpu, half):
    r = np.random.RandomState(1)
    x = r.randn(4, 33).astype(np.float32)
    t = np.array([0, 5, 32, 7])
    g = np.array([[7e4, 1e-8, 1 / 3, 0.0], [0.0, 0.0, 1 / 3, 7e4]], np.float32)
    logits = Tensor(N.DeviceArray.from_host(x), x.shape, requires_grad=True)
    logits._grad_dtype = np.float32
    nm.token_log_probs(logits, t).backward(g)
    want = R.logprobs_grad(x, t, g[0].astype(np.float64), g[1].astype(np.float64))
    got = logits.grad.reshape(x.shape).astype(np.float64)
    # per row: p and log p to (|log p| + 4)·2^-23 relative, both below 8 here
    for i in range(4):
        assert np.abs(got[i] - want[i]).max() <= (abs(g[0, i]) + 8 * abs(g[1, i])) * 12 * 2.0**-22, i


def test_upstream_gradients_of_float16_logits(gpu, half):
    """Logits of float16 beside a probability of nearly one: 7e4 times what is left is in range."""
    x = np.array([[8.0, 0.0, -1.0], [9.0, 1.0, 0.0]], np.float16)
    t, g = np.array([0, 0]), np.array([[7e4, -7e4], [0.0, 0.0]], np.float32)
    logits = Tensor(x, x.shape, requires_grad=True)
    nm.token_log_probs(logits, t).backward(g)
    want = R.logprobs_grad(x, t, g[0].astype(np.float64), np.zeros(2))
    got = np.asarray(logits.grad).reshape(x.shape).astype(np.float64)
    # p to (|log p| + 4)·2^-23 relative, |log p| < 10: at the target 7e4·p is taken from 7e4; then
    # half a step of float16
    assert np.abs(got - want).max() <= 7e4 * 14 * 2.0**-23 + np.abs(want).max() * 2.0**-11
