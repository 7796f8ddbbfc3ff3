"""The 4-bit cache and the token log probabilities refuse what they cannot run before anything
is launched (no GPU needed: the checks come first)."""
import ctypes as C

import numpy as np
import pytest

from nimbleml_amd import _native as N
from nimbleml_amd import kernels as K
from nimbleml_amd.gpt import check_kv_bits
from oracle import kv4_ref as R

P = 1 << 20  # a pointer that no call here may reach


def refused(fn, *args, match):
    with pytest.raises((RuntimeError, ValueError), match=match):
        N.check(fn(*args))


def write(batch=2, heads=2, seq=3, max_seq=8, dk=64, dtype=1, k=P, codes=P, stride=64):
    return (N.lib.nml_kv4_write_device, k, P, stride, stride, stride, codes, P, P, P, None, None,
            batch, heads, seq, max_seq, dk, None, dtype)


def read(batch=2, heads=2, seq=3, max_seq=8, dk=64, dtype=1, out=P):
    return (N.lib.nml_kv4_read_device, P, P, P, P, None, None, out, P, batch, heads, seq, max_seq,
            dk, None, dtype)


def attend(batch=2, heads=4, kv=2, seq=1, max_seq=8, dk=64, scale=8.0, lens=P, ws=16, nbytes=1 << 40,
           dtype=1):
    return (N.lib.nml_kv4_attention_device, P, P, P, P, P, lens, None, P, batch, heads, kv, seq,
            max_seq, dk, scale, ws, nbytes, None, dtype)


@pytest.mark.parametrize("call, match", [
    (write(dk=0), "head_dim"), (write(dk=257), "head_dim"), (write(dtype=2), "dtype"),
    (write(max_seq=0), "max_seq"), (write(max_seq=1 << 31), "max_seq"),
    (write(batch=1 << 16), "too many"), (write(heads=1 << 14, seq=1 << 13), "too many"),
    (write(k=None), "null"), (write(codes=None), "null"), (write(codes=P + 8), "aligned"), (write(stride=1 << 41), "stride"),
    (read(dk=300), "head_dim"), (read(out=None), "null"), (read(dtype=-1), "dtype"),
    (attend(heads=5), "divisible"), (attend(kv=0), "divisible"), (attend(scale=0.0), "scale_div"),
    (attend(scale=float("nan")), "scale_div"), (attend(lens=None), "null"),
    (attend(scale=1e-39), "normal"), (attend(scale=float("inf")), "normal"),
    (attend(batch=4096, heads=2048, kv=2048), "too many"),
    (attend(ws=24), "aligned"), (attend(max_seq=0), "max_seq"), (attend(dk=512), "head_dim"),
])
def test_kv4_refusals(call, match):
    refused(*call, match=match)


def test_kv4_nothing_to_do():
    for call in (write(batch=0), write(seq=0), read(heads=0), attend(seq=0), attend(batch=0)):
        N.check(call[0](*call[1:]))


def test_kv4_workspace_is_checked():
    need = C.c_size_t(7)
    N.check(N.lib.nml_kv4_attention_workspace(1, 16, 16, 1, 65536, 128, C.byref(need)))
    if need.value:
        refused(*attend(batch=1, heads=16, kv=16, max_seq=65536, dk=128, nbytes=need.value - 1),
                match="workspace")
        refused(*attend(batch=1, heads=16, kv=16, max_seq=65536, dk=128, ws=None), match="workspace")
    N.check(N.lib.nml_kv4_attention_workspace(0, 0, 0, 1, 1, 1, C.byref(need)))
    assert need.value == 0
    refused(N.lib.nml_kv4_attention_workspace, 1, 3, 2, 1, 1, 1, C.byref(need), match="divisible")
    refused(N.lib.nml_kv4_attention_workspace, 1, 2, 2, 1, 1, 1, None, match="null")


def score(rows=2, vocab=50, ld=50, top_k=0, logits=P, targets=P, logp=P, ids=None, dtype=0):
    return (N.lib.nml_token_logprobs_device, logits, ld, targets, rows, vocab, 0, 0, top_k, logp,
            None, None, None, ids, None, None, dtype)


def grad(rows=2, vocab=50, ld=50, ld_d=50, m=P, l=P, entropy=None, dentropy=None, dtype=0):
    return (N.lib.nml_token_logprobs_backward_device, P, ld, P, m, l, entropy, None, dentropy, rows,
            vocab, 0, 0, P, ld_d, None, dtype)


@pytest.mark.parametrize("call, match", [
    (score(vocab=0, ld=0), "out of range"), (score(ld=49), "out of range"), (score(dtype=7), "dtype"),
    (score(top_k=51), "top_k"), (score(vocab=1000, ld=1000, top_k=65), "top_k"),
    (score(top_k=3), "top_ids"), (score(logits=None), "null"), (score(targets=None), "targets"),
    (grad(ld=3), "out of range"), (grad(ld_d=3), "out of range"), (grad(m=None), "null"), (grad(l=None), "null"),
    (grad(dentropy=P), "entropy"), (grad(dtype=3), "dtype"),
])
def test_logprobs_refusals(call, match):
    refused(*call, match=match)


def test_logprobs_nothing_to_do():
    N.check(score(rows=0)[0](*score(rows=0)[1:]))
    N.check(grad(rows=0)[0](*grad(rows=0)[1:]))


def test_python_refusals():
    x, y = np.zeros((2, 7), np.float32), np.zeros(2, np.int64)
    for k in (-1, 65):
        with pytest.raises(ValueError, match="top_k"):
            K.token_logprobs(x, y, k)
    for bits in (8, 16, 0, "4"):
        with pytest.raises(ValueError, match="kv_bits"):
            check_kv_bits(bits)


def test_models_that_are_not_there():
    out = C.c_void_p(5)
    refused(N.lib.nml_cache_create_kv4, None, 1, C.byref(out), match="null")
    assert not out.value
    refused(N.lib.nml_model_logprobs, None, P, P, 1, 1, 0, 0, 0, P, P, None, None, match="null")


def test_oracle_rounds_to_the_nearest_code():
    """Held values are the nearest representable ones, and a held vector holds itself."""
    r = np.random.RandomState(0)
    for dt in (np.float16, np.float32):
        x = (r.randn(40, 3, 77) * 2.0 ** r.randint(-18, 10, (40, 3, 1))).astype(dt)
        codes, scales = R.quantise(x)
        y = R.values(codes, scales, 77)
        step = 2.0 ** (np.repeat(scales, 32, -1)[..., :77].astype(np.float64) - 127)
        grid = np.concatenate([R.GRID, -R.GRID])
        best = np.abs(x.astype(np.float64)[..., None] - grid * step[..., None]).min(-1)
        assert np.array_equal(np.abs(y - x), best)
        # every block's largest value is at least half of the largest code, so the scale is tight
        assert (np.abs(x).max() == 0) or np.abs(y).max() > 0
        assert np.array_equal(R.held(y.astype(dt)), y)
