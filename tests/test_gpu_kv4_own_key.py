"""A decode step over a 4-bit cache takes its own key and value, which its attention codes and writes:
a model in which a token's own key decides its output, so that one left out, or bytes written
otherwise, change the logits by much."""
import numpy as np
import pytest

import nimbleml_amd as nm
from oracle import kv4_ref as Q
from oracle.weights import GPTConfig, make_weights

pytestmark = pytest.mark.gpu

STEPS = (95, 94)  # tokens that the prompts do not hold


def decisive(cfg, dtype):
    """One layer whose q, k and v are the normalised token itself (q and k times 4), no positions, no
    feed-forward; tokens of ±1 and ±0.6, sixteen of each in a block of 32 (eight in one of 16)."""
    r = np.random.RandomState(cfg.d_model)
    w = {n: np.zeros_like(a) if not n.endswith("gamma") else np.ones_like(a)
         for n, a in make_weights(cfg, seed=1, dtype=dtype).items()}
    e = np.empty((cfg.vocab_size, cfg.d_model))
    for t in range(cfg.vocab_size):
        for h in range(0, cfg.d_model, cfg.head_dim):
            for at in range(0, cfg.head_dim, 32):
                n = min(32, cfg.head_dim - at)
                e[t, h + at:h + at + n] = r.permutation(np.tile([1.0, 0.6], n // 2)) * r.choice([-1, 1], n)
    w["token_emb.weights"] = e.astype(dtype)
    for name, a in (("W_q", 4.0), ("W_k", 4.0), ("W_v", 1.0), ("W_o", 1.0)):
        w[f"blocks.layers.0.mha.{name}.weights"] = (a * np.eye(cfg.d_model)).astype(dtype)
    return w, w["token_emb.weights"].astype(np.float64)


def expected(cfg, e, prompt, token, dtype, own=True):
    """Logits of `token` after `prompt` by the formulas in 64 bits (own=False: its key left out)."""
    x = e[list(prompt) + [token]]
    n = x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-5)
    heads = n.reshape(len(n), cfg.num_heads, cfg.head_dim).transpose(1, 0, 2)
    kv = np.ascontiguousarray(heads).astype(dtype)
    k, v = Q.held(4 * kv), Q.held(kv)
    s = k @ (4 * heads[:, -1, :, None]) / np.sqrt(cfg.head_dim)
    if not own:
        s[:, -1] = -np.inf
    p = np.exp(s - s.max(1, keepdims=True))
    h = x[-1] + ((p / p.sum(1, keepdims=True)) * v).sum(1).reshape(-1)
    return h / np.sqrt((h * h).mean() + 1e-5) @ e.T


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("d, heads", [(64, 2), (64, 1), (160, 2), (128, 1), (256, 1)])
@pytest.mark.parametrize("batch", [1, 3])
def test_a_step_attends_to_its_own_key(gpu, dtype, d, heads, batch):
    cfg = GPTConfig(96, d, heads, 1, 4700)
    w, e = decisive(cfg, dtype)
    m = nm.GPT.from_arrays(w, 96, d, heads, 1, 4700, dtype=dtype)
    r = np.random.RandomState(d)
    # normalised values are 5e-6 (float32: 1e-7) relative from e / √0.68, codes' borders 3 %; the
    # head sums d products of size 1.3 in the dtype's accumulation, attention as in its own tests:
    # in float16 a few roundings of values of size 2, each entering d products
    tol = d * (2.0**-17 if dtype == np.float32 else 2.0**-8)
    lengths = (1, 30, 31, 32, 255, 256, 511, 512, 1023, 1024, 2047, 2048, 4095, 4096, 4510, 4607)
    for n in lengths if batch == 1 else lengths[2::4]:
        ids = r.randint(0, 94, (batch, n))
        step = np.tile(np.array(STEPS)[None], (batch, 1))
        _, a = m.forward_with_cache(ids, kv_bits=4)
        for t in range(2):
            got = m.forward_with_cache(step[:, t:t + 1], a)[0].numpy()[:, 0].astype(np.float64)
            for b in range(batch):
                before = list(ids[b]) + list(STEPS[:t])
                want = expected(cfg, e, before, STEPS[t], dtype)
                lost = expected(cfg, e, before, STEPS[t], dtype, own=False)
                assert np.abs(lost - want).max() > 8 * tol  # (the case can tell)
                assert np.abs(got[b] - want).max() <= tol, (n, t, b)
        # the same two written by one call of two tokens: q, k and v are exact multiples of one value,
        # so the bytes are equal and what attends to them is bit for bit
        _, c = m.forward_with_cache(ids, kv_bits=4)
        m.forward_with_cache(step, c)
        assert np.array_equal(m.forward_with_cache(step, a)[0].numpy(), m.forward_with_cache(step, c)[0].numpy()), n


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("d, heads", [(64, 2), (128, 1)])
def test_steps_after_ragged_prompts(gpu, dtype, d, heads):
    """Rows of one batch at different edges, a long one among them."""
    cfg = GPTConfig(96, d, heads, 1, 4700)
    w, e = decisive(cfg, dtype)
    m = nm.GPT.from_arrays(w, 96, d, heads, 1, 4700, dtype=dtype)
    r = np.random.RandomState(d + 1)
    rows = [r.randint(0, 94, n) for n in (31, 4095, 255, 1, 256, 2047)]
    _, cache = m.prefill_ragged(rows, kv_bits=4)
    tol = d * (2.0**-17 if dtype == np.float32 else 2.0**-8)
    for t in range(2):
        got = m.forward_with_cache(np.full((6, 1), STEPS[t]), cache)[0].numpy()[:, 0].astype(np.float64)
        for b, row in enumerate(rows):
            want = expected(cfg, e, list(row) + list(STEPS[:t]), STEPS[t], dtype)
            assert np.abs(got[b] - want).max() <= tol, (t, b)
