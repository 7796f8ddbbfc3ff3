"""distill_loss takes its teacher's entries as lists, arrays and Tensors alike."""
import numpy as np
import pytest

import nimbleml_amd as nm
from nimbleml_amd import _native as N

pytestmark = pytest.mark.gpu


def test_entries_in_every_form(gpu):
    r = np.random.RandomState(0)
    ids, top = r.randint(-1, 30, (2, 3, 4)), r.randn(2, 3, 4).astype(np.float32)
    x, grad = r.randn(2, 3, 30), r.randn(2, 3)
    got = []
    for i, y in ((ids, top), (ids.tolist(), top.tolist()), (nm.Tensor.from_int64(ids, ids.shape), nm.Tensor(top, top.shape)),
                 (N.DeviceArray.from_host(ids), N.DeviceArray.from_host(top))):
        logits = nm.Tensor(x, x.shape, requires_grad=True)
        loss = nm.distill_loss(logits, i, y, temperature=1.5)
        loss.backward(grad)
        got.append((np.asarray(loss.data), logits.grad))
    for loss, g in got[1:]:
        assert np.array_equal(loss, got[0][0]) and np.array_equal(g, got[0][1])
