"""The 4-bit cache and the token log probabilities in the model's own paths: cached forwards,
prompts of one length and of several, generate, scoring and its gradient through the model."""
import numpy as np
import pytest

import nimbleml_amd as nm
from nimbleml_amd import _native as N
from oracle import gpt_ref as R
from oracle import grad_ref as G
from oracle import kv4_ref as Q
from oracle.weights import GPTConfig, make_weights, random_ids

pytestmark = pytest.mark.gpu

CFG = GPTConfig(97, 48, 3, 2, 40)  # head dim 16


def model(w, cfg, dtype, rope=False):
    return nm.GPT.from_arrays(w, cfg.vocab_size, cfg.d_model, cfg.num_heads, cfg.num_layers,
                              cfg.max_seq_len, dtype=dtype, **({"use_rope": True} if rope else {}))


class Held:
    """The oracle with attention over the values that a 4-bit cache holds of K and V. `near`: the
    least distance of a K or V from where its code would change, as a share of the value."""

    def __init__(self, monkeypatch):
        self.near = np.inf
        plain = R.sdpa

        def sdpa(q, k, v, scale, mask):
            for x in (k, v):
                self.look(x)
            return plain(q, *(Q.held(x).astype(x.dtype) for x in (k, v)), scale, mask)

        monkeypatch.setattr(R, "sdpa", sdpa)

    def look(self, x):
        _, scales = Q.quantise(x)
        step = 2.0 ** (np.repeat(scales, 32, -1)[..., :x.shape[-1]].astype(np.float64) - 127)
        a = np.abs(x) / step
        mids = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
        self.near = min(self.near, (np.abs(a[..., None] - mids) / mids).min())
        pad = np.zeros(x.shape[:-1] + (-x.shape[-1] % 32,))
        top = np.abs(np.concatenate([x, pad], -1)).reshape(x.shape[:-1] + (-1, 32)).max(-1)
        edge = 1.75 * 2.0 ** np.floor(np.log2(top))  # where the scale changes, as at the next power
        self.near = min(self.near, (np.abs(top / edge - 1)).min(), (np.abs(top / (edge / 1.75) - 1)).min())


@pytest.mark.parametrize("rope", [False, True])
def test_cached_forwards_match_the_oracle_over_held_values(gpu, monkeypatch, rope):
    """float32: a prompt, then pieces of several tokens, then single ones; every position's logits
    against the oracle's forward with K and V replaced by what the cache holds of them."""
    from oracle.weights import rope_weights

    w = make_weights(CFG, seed=11, dtype=np.float32, rich=True)
    cache_of_rope = None
    if rope:
        w = rope_weights(w)
        cache_of_rope = R.rope_cache(CFG.max_seq_len, CFG.head_dim)
    ids = random_ids((2, 33), CFG.vocab_size, seed=22)
    held = Held(monkeypatch)
    want = R.forward(w, ids, CFG.num_heads, CFG.num_layers, cache_of_rope)
    # float32 K and V here and there are within 1e-5 of each other: no code may lie nearer a border
    assert held.near > 1e-5, held.near
    m = model(w, CFG, np.float32, rope)
    for cuts in ([33], [20, 21, 22, 33], [5, 9, 25, 33], list(range(1, 34))):
        cache, got, at = None, [], 0
        for end in cuts:
            lg, cache = m.forward_with_cache(ids[:, at:end], cache, kv_bits=4)
            got.append(lg.numpy())
            at = end
        assert cache.length == 33 and cache.kv_bits == 4
        assert np.abs(np.concatenate(got, 1) - want).max() <= 1e-3, cuts


def test_ragged_prompts_and_steps(gpu):
    """Rows of different lengths in one pass, then one token each: as each row alone."""
    w = make_weights(CFG, seed=12, dtype=np.float32, rich=True)
    m = model(w, CFG, np.float32)
    rows = [random_ids((n,), CFG.vocab_size, seed=n) for n in (7, 30, 1, 18)]
    step = random_ids((4, 2), CFG.vocab_size, seed=99)
    lg, cache = m.prefill_ragged(rows, kv_bits=4)
    first = lg.numpy()
    nxt = [m.forward_with_cache(step[:, i:i + 1], cache)[0].numpy() for i in range(2)]
    for b, row in enumerate(rows):
        a, c = m.forward_with_cache(row[None], kv_bits=4)
        assert np.abs(a.numpy()[0, -1] - first[b]).max() <= 1e-3
        for i in range(2):
            a, c = m.forward_with_cache(step[b:b + 1, i:i + 1], c)
            assert np.abs(a.numpy()[0, -1] - nxt[i][b, -1]).max() <= 1e-3


@pytest.mark.parametrize("piece", [2, 16, 17, 25])
def test_pieces_after_ragged_prompts(gpu, piece):
    """Several tokens a row from different positions on, attended to in place and read back."""
    w = make_weights(CFG, seed=15, dtype=np.float32, rich=True)
    m = model(w, CFG, np.float32)
    rows = [random_ids((n,), CFG.vocab_size, seed=n) for n in (7, 13, 1, 10)]
    more = random_ids((4, piece), CFG.vocab_size, seed=98)
    _, cache = m.prefill_ragged(rows, kv_bits=4)
    got = m.forward_with_cache(more, cache)[0].numpy()
    after = m.forward_with_cache(more[:, :1], cache)[0].numpy()
    for b, row in enumerate(rows):
        _, c = m.forward_with_cache(row[None], kv_bits=4)
        want = m.forward_with_cache(more[b:b + 1], c)[0].numpy()
        assert np.abs(want[0] - got[b]).max() <= 1e-3
        want = m.forward_with_cache(more[b:b + 1, :1], c)[0].numpy()
        assert np.abs(want[0] - after[b]).max() <= 1e-3


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("batch, graph", [(1, True), (3, False), (16, True)])
def test_generate_is_the_argmax_of_cached_forwards(gpu, dtype, batch, graph):
    """Greedy generate over a 4-bit cache (graph replay, and the two-stream step at batch 16)
    against the same tokens fed one by one: at each step the chosen token's logit is within the
    dtype's rounding of the largest."""
    w = make_weights(CFG, seed=13, dtype=dtype, rich=True)
    m = model(w, CFG, dtype)
    ids = random_ids((batch, 9), CFG.vocab_size, seed=5)
    out = nm.generate(m, ids, max_new_tokens=20, temperature=0.0, kv_bits=4, use_graph=graph)
    assert np.array_equal(out[:, :9], ids)
    again = nm.generate(m, ids, max_new_tokens=20, temperature=0.0, kv_bits=4, use_graph=graph)
    assert np.array_equal(out, again)
    lg, cache = m.forward_with_cache(ids, kv_bits=4)
    lg = lg.numpy()[:, -1].astype(np.float64)
    tol = 1e-3 if dtype == np.float32 else 3e-2
    for t in range(9, 29):
        chosen = np.take_along_axis(lg, out[:, t:t + 1], 1)[:, 0]
        assert (lg.max(1) - chosen <= tol).all(), t
        if t < 28:
            lg = m.forward_with_cache(out[:, t:t + 1], cache)[0].numpy()[:, -1].astype(np.float64)


def test_four_bits_change_little_and_something(gpu):
    """The same prompt over both caches: logits differ (the values are rounded) and by no more than
    a step of 4 bits can move them here."""
    w = make_weights(CFG, seed=14, dtype=np.float32, rich=True)
    m = model(w, CFG, np.float32)
    ids = random_ids((2, 30), CFG.vocab_size, seed=6)
    a = m.forward_with_cache(ids)[0].numpy()
    b = m.forward_with_cache(ids, kv_bits=4)[0].numpy()
    assert 0 < np.abs(a - b).max() < 0.2 * np.abs(a).max()


def test_kv_bits_are_checked(gpu):
    m = model(make_weights(CFG, seed=1, dtype=np.float32), CFG, np.float32)
    ids = random_ids((1, 4), CFG.vocab_size, seed=1)
    for bad in (8, 0, 16, "4"):
        with pytest.raises(ValueError, match="kv_bits"):
            m.forward_with_cache(ids, kv_bits=bad)
        with pytest.raises(ValueError, match="kv_bits"):
            nm.generate(m, ids, max_new_tokens=2, kv_bits=bad)
        with pytest.raises(ValueError, match="kv_bits"):
            m.prefill_ragged([ids[0]], kv_bits=bad)
    with pytest.raises(ValueError, match="use_kv_cache"):
        nm.generate(m, ids, max_new_tokens=2, kv_bits=4, use_kv_cache=False)
    _, cache = m.forward_with_cache(ids)
    with pytest.raises(ValueError, match="kv_bits"):
        m.forward_with_cache(ids, cache, kv_bits=4)
    with pytest.raises(ValueError, match="exceeds maximum sequence length"):
        m.forward_with_cache(random_ids((1, 41), CFG.vocab_size, seed=1), kv_bits=4)


# ------------------------------------------------------------------------ scoring

@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_scores_of_the_model(gpu, dtype):
    w = make_weights(CFG, seed=15, dtype=dtype, rich=True)
    m = model(w, CFG, dtype)
    ids, lab = (random_ids((3, 21), CFG.vocab_size, seed=s) for s in (7, 8))
    lab[1, 4:] = -100
    got = m.log_probs(ids, lab, top_k=5, ignore_index=-100)
    lg = m.forward(ids).numpy().reshape(63, -1)
    want = Q.logprobs(lg, lab.reshape(-1), 5, -100)
    # the same logits: only the statistics' float32
    assert np.abs(got["logp"].numpy().reshape(-1) - want[0]).max() <= 1e-5
    assert np.abs(got["entropy"].numpy().reshape(-1) - want[1]).max() <= 1e-5
    assert np.array_equal(got["top_ids"].numpy().reshape(63, 5), want[4])
    assert np.abs(got["top_logp"].numpy().reshape(63, 5) - want[5]).max() <= 1e-5
    with nm.no_grad():
        loss = m.compute_loss(ids, lab, ignore_index=-100).item()
    kept = lab.reshape(-1) != -100
    tol = 1e-5 if dtype == np.float32 else 2e-2  # the float16 loss rounds its exponentials
    assert abs(-got["logp"].numpy().reshape(-1)[kept].mean() - loss) <= tol
    with pytest.raises(ValueError, match="out of range"):
        m.log_probs(ids, np.full((3, 21), 97), top_k=0)
    with pytest.raises(ValueError, match="label count"):
        m.log_probs(ids, lab[:, :-1])


def test_gradients_through_the_model(gpu):
    """token_log_probs over forward's logits: with −1/n on every log probability the parameters'
    gradients are compute_loss's, checked against the float64 gradient oracle; an entropy's
    gradient against differences of the oracle's."""
    CFG = GPTConfig(96, 48, 3, 2, 40)  # the backward's products take multiples of 4
    w = make_weights(CFG, seed=16, dtype=np.float32, rich=True)
    m = model(w, CFG, np.float32)
    ids, lab = (random_ids((2, 11), CFG.vocab_size, seed=s) for s in (9, 10))
    out = nm.token_log_probs(m.forward(ids), lab)
    assert out.shape == (2, 2, 11)
    g = np.zeros(out.shape, np.float32)
    g[0] = -1.0 / lab.size
    out.backward(g)
    w64 = {k: v.astype(np.float64) for k, v in w.items()}
    _, grads = G.loss_and_grads(w64, ids, lab, CFG.num_heads, CFG.num_layers)
    for name, p in nm.named_parameters(m):
        want = grads[name]
        err = np.abs(np.asarray(p.grad, np.float64).reshape(want.shape) - want).max()
        assert err <= 1e-4 * max(np.abs(want).max(), 1e-3), name
    # entropy, along one direction of one parameter
    for _, p in nm.named_parameters(m):
        p.zero_grad()
    g[:] = 0.0
    g[1] = 1.0
    nm.token_log_probs(m.forward(ids), lab).backward(g)
    got = {n: np.asarray(p.grad, np.float64) for n, p in nm.named_parameters(m)}

    def total(name, d, h):
        v = dict(w64)
        v[name] = v[name] + h * d
        lg = R.forward(v, ids, CFG.num_heads, CFG.num_layers).reshape(lab.size, -1)
        return Q.logprobs(lg, lab.reshape(-1))[1].sum()

    r = np.random.RandomState(0)
    for name in ("token_emb.weights", "blocks.layers.1.mha.W_q.weights", "ln.gamma"):
        d = r.randn(*w64[name].shape)
        d /= np.linalg.norm(d)
        h = 1e-4
        slope = (total(name, d, h) - total(name, d, -h)) / (2 * h)
        along = float((got[name].reshape(d.shape) * d).sum())
        # differences: h²·f''' / 6 and 1e-16·f / h, both below 1e-6; float32 gradients 1e-4 relative
        assert abs(along - slope) <= 1e-4 * np.linalg.norm(got[name]) + 1e-5, name


def test_no_gradient_under_no_grad(gpu):
    m = model(make_weights(CFG, seed=1, dtype=np.float32), CFG, np.float32)
    ids = random_ids((1, 5), CFG.vocab_size, seed=1)
    with nm.no_grad():
        out = nm.token_log_probs(m.forward(ids), ids)
    assert not out.requires_grad and out._backward is None


def test_a_piece_reads_back_what_steps_wrote(gpu):
    """Fourteen single tokens and the other nineteen at once, as the whole at once."""
    m = model(make_weights(CFG, seed=11, dtype=np.float32, rich=True), CFG, np.float32)
    ids = random_ids((2, 33), CFG.vocab_size, seed=22)
    want = m.forward_with_cache(ids, kv_bits=4)[0].numpy()
    cache = None
    for t in range(14):
        _, cache = m.forward_with_cache(ids[:, t:t + 1], cache, kv_bits=4)
    assert np.abs(m.forward_with_cache(ids[:, 14:], cache)[0].numpy() - want[:, 14:]).max() <= 1e-3


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("d, heads", [(64, 2), (64, 1), (160, 2), (128, 1), (256, 1)])
def test_steps_over_long_rows(gpu, dtype, d, heads):
    """Two single tokens after prompts that end at a tile's, a wave's and a piece's edge, as both in
    one call: the step's own key is the last of a tile, the first of one, of a piece."""
    cfg = GPTConfig(96, d, 1, heads, 4700)
    m = model(make_weights(cfg, seed=16, dtype=dtype, rich=True), cfg, dtype)
    tol = 1e-3 if dtype == np.float32 else 3e-2
    for n in (1, 31, 32, 255, 256, 2047, 2048, 4096, 4510, 4607):
        ids = random_ids((3, n + 2), cfg.vocab_size, seed=n)
        _, a = m.forward_with_cache(ids[:, :n], kv_bits=4)
        want = m.forward_with_cache(ids[:, n:], a)[0].numpy().astype(np.float64)
        _, b = m.forward_with_cache(ids[:, :n], kv_bits=4)
        for t in range(2):
            got = m.forward_with_cache(ids[:, n + t:n + t + 1], b)[0].numpy().astype(np.float64)
            assert np.abs(got[:, 0] - want[:, t]).max() <= tol, (n, t)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_scoring_and_decoding_between_a_loss_and_its_backward(gpu, dtype):
    """Neither touches what the loss keeps for its backward: the gradients are bit for bit those
    without them (the training path sums in a fixed order)."""
    cfg = GPTConfig(96, 48, 3, 2, 40)
    w = make_weights(cfg, seed=17, dtype=dtype, rich=True)
    ids, lab = (random_ids((2, 12), cfg.vocab_size, seed=s) for s in (3, 4))
    grads = []
    for between in (False, True):
        m = model(w, cfg, dtype)
        loss = m.compute_loss(ids, lab)
        if between:
            other = random_ids((3, 30), cfg.vocab_size, seed=5)
            m.log_probs(other, other, top_k=3)
            nm.generate(m, other, max_new_tokens=4, temperature=0.0, kv_bits=4)
        loss.backward()
        grads.append({n: np.asarray(p.grad) for n, p in nm.named_parameters(m)})
    for name in grads[0]:
        assert np.array_equal(grads[0][name], grads[1][name]), name
