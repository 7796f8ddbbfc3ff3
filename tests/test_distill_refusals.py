"""Distillation in place (no GPU needed: the checks come first)."""
import pytest

from nimbleml_amd import _native as N

P = 1 << 20  # a pointer that no call here may reach


def test_a_gradient_in_place_keeps_the_logits_stride():
    """At another stride a row's gradient would lie over logits of rows that are still to be read."""
    for ld, ld_d in ((128, 100), (100, 128)):
        with pytest.raises(RuntimeError, match="in place"):
            N.check(N.lib.nml_distill_backward_device(P, ld, P, P, P, P, P, 4, 100, 8, 1.0, P, ld_d, None, 0))
