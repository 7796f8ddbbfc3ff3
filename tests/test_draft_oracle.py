"""The 64-bit statements of oracle/draft_ref.py against differences and against each other, and the
refusals of the operators that they state (no GPU needed: the checks come first)."""
import ctypes as C

import numpy as np
import pytest

from nimbleml_amd import _native as N
from nimbleml_amd import kernels as K
from oracle import draft_ref as R

P = 1 << 20  # a pointer that no call here may reach


def refused(fn, *args, match):
    with pytest.raises((RuntimeError, ValueError), match=match):
        N.check(fn(*args))


def test_distill_gradient_against_differences():
    r = np.random.RandomState(0)
    x, y = r.randn(3, 17) * 2, r.randn(3, 5).astype(np.float32) * 2
    ids = np.array([[0, 3, 3, 16, -1], [-1] * 5, [1, 2, 4, 5, 6]])
    dloss, t, h = r.randn(3), 1.7, 1e-5
    grad, _, _ = R.distill_grad(x, ids, y, dloss, t)
    for i in range(3):
        for v in range(17):
            a, b = x.copy(), x.copy()
            a[i, v] += h
            b[i, v] -= h
            diff = (R.distill(a, ids, y, t)[0] - R.distill(b, ids, y, t)[0]) @ dloss / (2 * h)
            # (the difference is off by h²/6 times a third derivative of order 1, and by 2^-53/h)
            assert abs(diff - grad[i, v]) < 1e-9


def test_verify_keeps_the_targets_distribution():
    """Of one draft from q, by the formula and not by sampling: P(token) = p."""
    r = np.random.RandomState(1)
    logits, draft = r.randn(2, 9), r.randn(9)
    p, q = np.exp(R.log_softmax(logits[0], 1.0)), np.exp(R.log_softmax(draft, 1.0))
    first = np.zeros(9)
    for d in range(9):
        ok = min(1.0, p[d] / q[d])
        first[d] += q[d] * ok
        left = np.maximum(p - q, 0)
        first += q[d] * (1 - ok) * left / left.sum()
    assert np.allclose(first, p, atol=1e-14)
    # and the oracle follows that rule on either side of the border
    d = int(np.argmax(q - p))
    border = p[d] / q[d]
    for u, want in ((border * (1 - 1e-9), 1), (border * (1 + 1e-9), 0)):
        got, _ = R.verify(logits[None], np.array([[d]]), np.array([[u, 0.5]]), draft[None, None], [1], 1.0)
        assert got[0] == want


def distill(rows=4, vocab=100, ld=100, top_k=8, t=1.0, logits=P, loss=P, dtype=0):
    return (N.lib.nml_distill_device, logits, ld, P, P, rows, vocab, top_k, t, loss, None, None, None,
            dtype)


def distill_bwd(rows=4, vocab=100, ld=100, top_k=8, t=1.0, m=P, ld_d=100, dtype=0):
    return (N.lib.nml_distill_backward_device, P, ld, P, P, m, P, P, rows, vocab, top_k, t, P, ld_d,
            None, dtype)


@pytest.mark.parametrize("call, match", [
    (distill(dtype=2), "dtype"), (distill(top_k=0), "top_k"), (distill(top_k=257), "top_k"),
    (distill(vocab=0), "out of range"), (distill(ld=99), "out of range"), (distill(rows=1 << 31), "out of range"),
    (distill(t=0.0), "temperature"), (distill(t=-1.0), "temperature"), (distill(t=float("nan")), "temperature"),
    (distill(t=float("inf")), "temperature"), (distill(logits=None), "null"), (distill(loss=None), "null"),
    (distill_bwd(m=None), "null"), (distill_bwd(ld_d=99), "stride"), (distill_bwd(t=1e-7), "temperature"),
])
def test_distill_refusals(call, match):
    refused(*call, match=match)


def verify(batch=2, n=3, vocab=100, ld=100, ld_d=100, t=1.0, u=P, drafts=P, ws=16, nbytes=1 << 40, dtype=1):
    return (N.lib.nml_verify_drafts_device, P, ld, P, ld_d, drafts, None, u, batch, n, vocab, t, P, P, ws,
            nbytes, None, dtype)


@pytest.mark.parametrize("call, match", [
    (verify(dtype=5), "dtype"), (verify(n=64), "drafts"), (verify(vocab=0), "vocabulary"),
    (verify(vocab=(1 << 24) + 1, ld=1 << 25, ld_d=1 << 25), "vocabulary"), (verify(batch=65535), "too many"),
    (verify(batch=1 << 40), "too large"), (verify(ld=99), "stride"), (verify(ld_d=99), "stride"),
    (verify(t=1e-7), "temperature"), (verify(t=float("nan")), "temperature"), (verify(u=None), "null"),
    (verify(drafts=None), "null"), (verify(ws=None), "workspace"), (verify(nbytes=100), "workspace"),
    (verify(ws=24), "aligned"),
])
def test_verify_refusals(call, match):
    refused(*call, match=match)


def write(batch=2, heads=2, seq=3, pages=4, page=16, total=9, dk=64, stride=64, k=P, table=P, dtype=1):
    return (N.lib.nml_paged_write_device, k, P, stride, stride, stride, P, P, table, None, None, batch,
            heads, seq, pages, page, total, dk, None, dtype)


def attend(batch=2, heads=4, kv=2, seq=1, pages=4, page=16, total=9, dk=64, scale=8.0, lens=P, table=P,
           ws=16, nbytes=1 << 40, dtype=1):
    return (N.lib.nml_paged_attention_device, P, P, P, table, lens, None, P, batch, heads, kv, seq, pages,
            page, total, dk, scale, ws, nbytes, None, dtype)


@pytest.mark.parametrize("call, match", [
    (write(dk=0), "head_dim"), (write(dk=257), "head_dim"), (write(dtype=2), "dtype"),
    (write(page=24), "power of two"), (write(page=4), "power of two"), (write(page=2048), "power of two"),
    (write(page=0), "power of two"), (write(pages=0), "out of range"), (write(pages=1 << 40), "out of range"),
    (write(total=0), "out of range"), (write(total=1 << 31), "out of range"), (write(k=None), "null"),
    (write(table=None), "null"), (write(stride=1 << 41), "stride"), (write(batch=1 << 16), "too many"),
    (write(heads=1 << 12, seq=1 << 11), "too many"),
    (attend(batch=4096, heads=2048, kv=2048), "too many"), (attend(pages=1 << 26, page=16, seq=1000), "too many"),
    (attend(heads=5), "divisible"), (attend(kv=0), "divisible"), (attend(scale=0.0), "scale_div"),
    (attend(scale=float("nan")), "scale_div"), (attend(scale=1e-39), "normal"),
    (attend(scale=float("inf")), "normal"), (attend(lens=None), "null"), (attend(table=None), "null"),
    (attend(ws=24), "aligned"), (attend(page=12), "power of two"), (attend(dk=300), "head_dim"),
    (attend(pages=1 << 16, ws=None), "workspace"), (attend(pages=1 << 16, nbytes=64), "workspace"),
])
def test_paged_refusals(call, match):
    refused(*call, match=match)


def test_nothing_to_do():
    for call in (distill(rows=0), distill_bwd(rows=0), verify(batch=0), write(batch=0), write(seq=0),
                 attend(seq=0), attend(batch=0), attend(heads=0, kv=0)):
        N.check(call[0](*call[1:]))


def test_workspaces():
    need = C.c_size_t(7)
    for fn, args in ((N.lib.nml_verify_drafts_workspace, (0, 3, 100)),
                     (N.lib.nml_paged_attention_workspace, (1, 16, 16, 1, 1, 16, 64, 1))):
        N.check(fn(*args, C.byref(need)))
        assert need.value == 0
    N.check(N.lib.nml_verify_drafts_workspace(1, 3, 100, C.byref(need)))
    assert need.value > 0
    N.check(N.lib.nml_paged_attention_workspace(1, 16, 16, 1, 4096, 16, 128, 1, C.byref(need)))
    assert need.value > 0


def test_pages_are_checked_on_the_host():
    table = np.array([[3, 1, 99], [0, -1, 2]])
    K._check_pages("x", table, [32, 16], 16, 4)  # (entries past a row's positions are not looked at)
    K._check_pages("x", table, [0, -5], 16, 4)
    for lens, match in (([33, 16], "page 99"), ([1, 17], "page -1"), ([49, 0], "needs 4 pages")):
        with pytest.raises(ValueError, match=match):
            K._check_pages("x", table, lens, 16, 4)


def test_wrappers_check_before_they_touch_the_device():
    x = np.zeros((2, 4, 10), np.float32)
    with pytest.raises(ValueError, match="uniforms are required"):
        K.verify_drafts(x, np.zeros((2, 3)))
    with pytest.raises(ValueError, match="drafts must be"):
        K.verify_drafts(x, np.zeros((2, 4)), temperature=0.0)
    with pytest.raises(ValueError, match="draft_logits must be"):
        K.verify_drafts(x, np.zeros((2, 3)), np.zeros((2, 4)), draft_logits=x)
    for empty in (np.zeros((2, 0), np.float32), np.float32(1)):
        with pytest.raises(ValueError, match="logits must be"):
            K.distill(empty, np.zeros((2, 3)), np.zeros((2, 3)))
    with pytest.raises(ValueError, match="power of two"):
        K.PagedKVCache(4, 24, 1, 64)
