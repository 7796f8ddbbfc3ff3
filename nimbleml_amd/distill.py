"""Distillation from a teacher's top logits with autograd.

The reference's loss knows one token a row (NimbleML/losses/cross_entropy.py:109-192); here the target
is what a teacher knows of its best tokens, such as ``GPT.log_probs``' alternatives: how a small model
learns to draft for a large one.
"""
from __future__ import annotations

import numpy as np

from nimbleml_amd import _native as N
from nimbleml_amd import kernels as K
from nimbleml_amd.grad_mode import is_grad_enabled
from nimbleml_amd.tensor import Tensor


def distill_loss(logits, top_ids, top_logits, *, temperature=1.0):
    """A float32 Tensor (*rows) of KL(q || p) for each row of ``logits`` (a Tensor (*rows, vocab), such
    as ``GPT.forward``'s): p its softmax at ``temperature``, q that of the teacher's ``top_logits``
    (*rows, k), logits or log probabilities, of the tokens ``top_ids`` (*rows, k). Ids of −1 are
    absent; rows of nothing else give 0. Not multiplied by temperature².

    With gradients wanted, ``backward(grad)`` with ``grad`` of the rows' shape adds the gradient of
    Σ grad·output to ``logits.grad`` (in the logits' dtype: float16 ones want the loss scaled, as
    ``compute_loss`` does) and goes on through the graph that made the logits."""
    rows = logits.shape[:-1]
    x = logits.data if isinstance(logits.data, N.DeviceArray) else \
        N.DeviceArray.from_host(np.asarray(logits.data))
    x = x.reshape(logits.shape)
    ids, top = (a if isinstance(a, N.DeviceArray) else N.DeviceArray.from_host(
        np.asarray(a.data, dtype=dt).reshape(a.shape) if isinstance(a, Tensor) else np.asarray(a, dtype=dt))
        for a, dt in ((top_ids, np.int64), (top_logits, np.float32)))
    loss, m, lsum = K.distill(x, ids, top, temperature)
    needs = is_grad_enabled() and logits.requires_grad
    out = Tensor(loss, rows, requires_grad=needs, _children=(logits,) if needs else ())
    out._grad_dtype = np.float32
    if needs:
        def _backward():
            if out.grad is None:
                return
            dloss = N.DeviceArray.from_host(np.asarray(out.grad, dtype=np.float32).reshape(-1))
            logits._accumulate_grad(K.distill_backward(x, ids, top, m, lsum, dloss,
                                                       temperature).numpy())

        out._backward = _backward
    return out
