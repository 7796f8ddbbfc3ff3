"""64-bit statements of the 4-bit KV cache and of token log probabilities.

The block format is the OCP microscaling one with E2M1 elements (blocks of 32, a power-of-two
scale); the choice of the scale is this framework's own (include/nimbleml_hip.h).
"""
import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
MIN_EXP = -120


def quantise(x):
    """(codes uint8 (..., blocks, 16), scales uint8 (..., blocks)) of x (..., dk)."""
    top = 13 if x.dtype == np.float16 else 125
    dk = x.shape[-1]
    nb = -(-dk // 32)
    w = np.zeros(x.shape[:-1] + (nb * 32,))
    w[..., :dk] = x
    w = w.reshape(x.shape[:-1] + (nb, 32))
    amax = np.abs(w).max(-1)
    finite = np.isfinite(amax)
    m, k = np.frexp(np.where(finite, amax, 0.0))  # amax = m·2^k with m in [½, 1)
    e = np.clip(np.where(m == 0, MIN_EXP, k - 3 + (m >= 0.875)), MIN_EXP, top)
    a = np.abs(np.where(finite[..., None], w, 0.0)) / 2.0 ** e[..., None]
    dist = np.abs(np.minimum(a, 6.0)[..., None] - GRID)
    low = dist.argmin(-1)  # of two as near, the lower …
    tie = (low < 7) & (np.take_along_axis(dist, low[..., None], -1)[..., 0] ==
                       np.take_along_axis(dist, np.minimum(low + 1, 7)[..., None], -1)[..., 0])
    c = low + (tie & (low % 2 == 1))  # … unless the upper one is even
    c = np.where(finite[..., None], c + 8 * np.signbit(w), 0).astype(np.uint8)
    return (c[..., 0::2] | (c[..., 1::2] << 4)), np.where(finite, e + 127, 255).astype(np.uint8)


def values(codes, scales, dk):
    """The float64 values (..., dk)."""
    c = np.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[:-1] + (32,))
    v = GRID[c & 7] * np.where(c & 8, -1.0, 1.0)
    e = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    v = v * e[..., None]
    return v.reshape(v.shape[:-2] + (-1,))[..., :dk]


def held(x):
    """The values the cache holds of x."""
    return values(*quantise(x), x.shape[-1])


def attention(q, k, v, lens, counts, scale):
    """q (b, heads, seq, dk) over the held k, v (b, kv_heads, max_seq, dk), float64; output
    (b, seq, heads·dk), zeros where a token sees no key or is past its row's count."""
    b, h, s, dk = q.shape
    g = h // k.shape[1]
    out = np.zeros((b, s, h, dk))
    for i in range(b):
        n = s if counts is None else int(counts[i])
        for t in range(n):
            keys = int(lens[i]) - n + t + 1
            if keys <= 0:
                continue
            for j in range(h):
                with np.errstate(invalid="ignore", over="ignore"):
                    x = k[i, j // g, :keys] @ q[i, j, t].astype(np.float64) / scale
                    p = np.exp(x - x.max())
                    out[i, t, j] = (p / p.sum()) @ v[i, j // g, :keys]
    return out.reshape(b, s, h * dk)


def logprobs(logits, targets, top_k=0, ignore_index=None):
    """(logp, entropy, m, l, top_ids, top_logp) in float64."""
    x = logits.astype(np.float64)
    with np.errstate(invalid="ignore", divide="ignore"):
        m = x.max(-1, keepdims=True)
        t = x - m
        z = np.exp(t).sum(-1)
        lp = t - np.log(z)[:, None]
        p = np.exp(lp)
        entropy = -np.where(p == 0, 0.0, p * np.where(p == 0, 0.0, lp)).sum(-1)
    logp = lp[np.arange(len(x)), np.clip(targets, 0, x.shape[1] - 1)]
    order = np.where(np.isnan(x), np.inf, x)
    nan_first = np.isnan(x)
    ids = np.stack([np.lexsort((np.arange(x.shape[1]), -order[r], ~nan_first[r]))[:top_k]
                    for r in range(len(x))]) if top_k else np.zeros((len(x), 0), np.int64)
    top = np.take_along_axis(lp, ids, -1)
    if ignore_index is not None:
        drop = targets == ignore_index
        logp, entropy, z = (np.where(drop, 0.0, a) for a in (logp, entropy, z))
        m = np.where(drop[:, None], 0.0, m)
        ids, top = np.where(drop[:, None], -1, ids), np.where(drop[:, None], 0.0, top)
    return logp, entropy, m[:, 0], z, ids, top


def logprobs_grad(logits, targets, dlogp, dentropy, ignore_index=None):
    """The gradient of Σ dlogp·logp + dentropy·entropy with respect to the logits."""
    x = logits.astype(np.float64)
    _, entropy, m, z, _, _ = logprobs(logits, targets)
    lp = x - m[:, None] - np.log(z)[:, None]
    p = np.exp(lp)
    hot = np.arange(x.shape[1]) == targets[:, None]
    d = dlogp[:, None] * (hot - p)
    d = d - dentropy[:, None] * p * np.where(p == 0, 0.0, np.where(p == 0, 0.0, lp) + entropy[:, None])
    return d if ignore_index is None else np.where((targets == ignore_index)[:, None], 0.0, d)
