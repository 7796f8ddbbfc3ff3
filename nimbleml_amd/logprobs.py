"""Log probabilities of tokens with autograd.

The reference averages them in its loss (NimbleML/losses/cross_entropy.py:109-192); here they are
kept row by row, so that a caller can weight them: a policy gradient, a preference loss over
answers, a distillation term, an entropy bonus.
"""
from __future__ import annotations

import numpy as np

from nimbleml_amd import _native as N
from nimbleml_amd import kernels as K
from nimbleml_amd.grad_mode import is_grad_enabled
from nimbleml_amd.tensor import Tensor


def token_log_probs(logits, targets, *, ignore_index=None):
    """A float32 Tensor (2, *rows) over the rows of ``logits`` (a Tensor (*rows, vocab), such as
    ``GPT.forward``'s): first the log probability of each row's target, then the entropy of its
    distribution; both 0 where the target is ``ignore_index``.

    With gradients wanted, ``backward(grad)`` with ``grad`` of that shape adds the gradient of
    Σ grad·output to ``logits.grad`` (in the logits' dtype: float16 ones want the loss scaled, as
    ``compute_loss`` does; ``grad`` itself is taken in float32) and goes on through the graph that
    made the logits. Logits of any vocabulary are scored and differentiated; the backward of a model
    (``GPT.forward``'s, as ``compute_loss``'s) takes vocabularies that are a multiple of 4 and raises
    for others."""
    rows = logits.shape[:-1]
    x = logits.data if isinstance(logits.data, N.DeviceArray) else \
        N.DeviceArray.from_host(np.asarray(logits.data))
    x = x.reshape(logits.shape)
    td = N.DeviceArray.from_host(np.asarray(
        targets.data if isinstance(targets, Tensor) else targets, dtype=np.int64).reshape(-1))
    logp, entropy, m, lsum, _, _ = K.token_logprobs(x, td, 0, ignore_index)
    both = N.DeviceArray((2, logp.size), np.float32)
    for i, part in enumerate((logp, entropy)):
        N.check(N.lib.nml_memcpy_d2d(both.ptr + i * part.nbytes, part.ptr, part.nbytes))
    needs = is_grad_enabled() and logits.requires_grad
    out = Tensor(both, (2, *rows), requires_grad=needs, _children=(logits,) if needs else ())
    out._grad_dtype = np.float32
    if needs:
        def _backward():
            if out.grad is None:
                return
            g = np.asarray(out.grad, dtype=np.float32).reshape(2, -1)
            dlogp, dentropy = (N.DeviceArray.from_host(g[i]) for i in range(2))
            logits._accumulate_grad(K.token_logprobs_backward(x, td, m, lsum, entropy, dlogp,
                                                              dentropy, ignore_index).numpy())

        out._backward = _backward
    return out
