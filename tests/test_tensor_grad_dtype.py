"""The upstream gradient that ``Tensor.backward`` is given arrives in the dtype that the tensor keeps
its gradient in: under float16 a float32 result's is not rounded to float16 on the way."""
import numpy as np
import pytest

import nimbleml_amd as nm
from nimbleml_amd import np_backend
from nimbleml_amd.tensor import Tensor

# past float16's range, below its least value, and with more bits than it has
UPSTREAM = np.array([7e4, 1e-8, 1 / 3, -0.0, 1.0], np.float32)


@pytest.fixture
def half():
    before = np_backend.dtype
    nm.set_dtype("float16")
    yield
    nm.set_dtype(np.dtype(before).name)


def seeded(x, grad, pinned):
    t = Tensor(x, (x.size,), requires_grad=True)
    if pinned:
        t._grad_dtype = np.float32
    seen = []
    t._backward = lambda: seen.append(t.grad.copy())
    t.backward(grad)
    return seen[0]


@pytest.mark.parametrize("kind", [np.asarray, np.float64, list])
def test_a_pinned_gradient_keeps_its_bits(half, kind):
    got = seeded(np.zeros(UPSTREAM.size), kind(UPSTREAM), True)
    assert got.dtype == np.float32 and np.array_equal(got, UPSTREAM)


@pytest.mark.parametrize("value", [7e4, 1e-8, 1 / 3])
def test_a_pinned_scalar_keeps_its_bits(half, value):
    got = seeded(np.zeros(1), value, True)
    assert got.dtype == np.float32 and got[0] == np.float32(value)


def test_other_gradients_are_in_the_compute_dtype(half):
    with np.errstate(over="ignore"):
        got = seeded(np.zeros(UPSTREAM.size), UPSTREAM, False)
        assert got.dtype == np.float16 and np.array_equal(got, UPSTREAM.astype(np.float16))
    assert seeded(np.zeros(1), None, False).dtype == np.float16
