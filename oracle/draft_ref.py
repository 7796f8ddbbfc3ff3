"""64-bit statements of distillation from a teacher's top logits, of the verification of drafted
tokens and of attention over a paged KV cache."""
import numpy as np


def teacher(ids, y, t):
    """(present (rows, k), q (rows, k)): the teacher's probabilities over a row's entries."""
    there = (ids >= 0) & (y > -np.inf)
    z = np.where(there, y.astype(np.float64) / t, -np.inf)
    top = np.where(there.any(-1), z.max(-1), 0.0)
    e = np.exp(z - top[:, None])
    return there, e / np.maximum(e.sum(-1, keepdims=True), 1e-300)


def log_softmax(x, t):
    x = x.astype(np.float64) / t
    m = x.max(-1, keepdims=True)
    return x - m - np.log(np.exp(x - m).sum(-1, keepdims=True))


def distill(x, ids, y, t):
    """(loss, m, l) of rows x (rows, vocab); rows without a teacher: zeros."""
    there, q = teacher(ids, y, t)
    lp = np.take_along_axis(log_softmax(x, t), np.maximum(ids, 0), -1)
    with np.errstate(divide="ignore", invalid="ignore"):
        terms = np.where(there & (q > 0), q * (np.log(q) - lp), 0.0)
    taught = there.any(-1)
    m = x.astype(np.float64).max(-1)
    l = np.exp((x.astype(np.float64) - m[:, None]) / t).sum(-1)
    return np.where(taught, terms.sum(-1), 0.0), np.where(taught, m, 0.0), np.where(taught, l, 0.0)


def distill_grad(x, ids, y, dloss, t):
    """d Σ dloss·loss / d x, and the probabilities p and q spread over the vocabulary."""
    there, q = teacher(ids, y, t)
    p = np.exp(log_softmax(x, t))
    spread = np.zeros_like(p)
    for r in range(x.shape[0]):
        np.add.at(spread[r], np.maximum(ids[r], 0), np.where(there[r], q[r], 0.0))
    d = (dloss.astype(np.float64) / t)[:, None] * (p - spread)
    return np.where(there.any(-1)[:, None], d, 0.0), p, spread


def verify(logits, drafts, u, draft_logits, counts, t):
    """(accepted (batch,), tokens (batch, n + 1)) of logits (batch, n + 1, vocab)."""
    batch, n1, vocab = logits.shape
    accepted = np.zeros(batch, np.int32)
    tokens = np.full((batch, n1), -1, np.int64)

    def dist(x):
        return np.exp(log_softmax(x, t))

    for b in range(batch):
        i = 0
        while True:
            if t <= 0:
                w = np.zeros(vocab)
                w[int(np.argmax(logits[b, i]))] = 1.0
            else:
                w = dist(logits[b, i])
            if i == counts[b]:
                break
            d = int(drafts[b, i])
            if t <= 0:
                if w[d] != 1.0:
                    break
            else:
                q = np.eye(1, vocab, d)[0] if draft_logits is None else dist(draft_logits[b, i])
                if not u[b, i] * q[d] < w[d]:
                    left = np.maximum(w - q, 0.0)
                    w = left if left.sum() > 0 else w
                    break
            tokens[b, i] = d
            i += 1
        accepted[b] = i
        if t <= 0:
            tokens[b, i] = int(np.argmax(w))
        else:
            run = np.cumsum(w)
            past = np.nonzero(run > u[b, -1] * run[-1])[0]
            tokens[b, i] = past[0] if len(past) else np.nonzero(w)[0][-1]
    return accepted, tokens


def gather_pages(pages, table, length):
    """(kv_heads, length, dk) of one row, in 64 bits."""
    size = pages.shape[2]
    ids = table[:-(-length // size)] if length else table[:0]
    x = np.concatenate(list(pages[ids].astype(np.float64)), 1) if len(ids) else \
        np.zeros((pages.shape[1], 0, pages.shape[3]))
    return x[:, :length]


def paged_attention(q, k_pages, v_pages, table, lens, counts, scale):
    """(out, its error's measure) of q (batch, heads, seq, dk), both (batch, seq, heads, dk): the
    second holds Σ p|v|, and as a third the largest Σ|q||k| / scale of any key of the row."""
    batch, heads, seq, dk = q.shape
    kv = k_pages.shape[1]
    out = np.zeros((batch, seq, heads, dk))
    size = np.zeros_like(out)
    spread = np.zeros((batch, seq, heads, 1))
    for b in range(batch):
        n, length = int(counts[b]), int(lens[b])
        k, v = gather_pages(k_pages, table[b], length), gather_pages(v_pages, table[b], length)
        for h in range(heads):
            for s in range(n):
                end = length - n + s + 1
                if end <= 0:
                    continue
                kk, vv, qq = k[h // (heads // kv), :end], v[h // (heads // kv), :end], q[b, h, s].astype(np.float64)
                x = kk @ qq / scale
                p = np.exp(x - x.max())
                p /= p.sum()
                out[b, s, h], size[b, s, h] = p @ vv, p @ np.abs(vv)
                spread[b, s, h] = (np.abs(kk) @ np.abs(qq)).max() / scale
    return out, size, spread
